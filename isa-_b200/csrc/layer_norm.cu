// layer_norm.cu — layer normalisation and its backward pass, alone and joined
// with the residual sum in front of it.
//
//   h = x + d (rounded to h's type; h = x without a branch d)
//   u = (h - mean(h)) * rstd,  rstd = (var(h) + eps)^-1/2,  y = u w + b
//   dx = rstd (g w - mean(g w) - u mean(g w u)) + dh,  dw = sum_rows g u,  db = sum_rows g
//
// Both directions are bound by HBM: every row is read once, the row sums are taken
// in registers (mean first, then the centred squares: no cancellation for rows far
// from zero), and the results leave in the same pass.  A row belongs to one to
// sixteen warps, so that a thread holds at most 16 elements of usual widths.  Rows
// come through shared memory by bulk copies, a ring of up to four per row group:
// enough bytes are under way whatever the registers allow (with the next row's
// loads held in registers the fp16 backward took 54 us at 50,432 x 384, not 33).
// The weight gradients are column sums: each thread keeps the sums of its own
// columns over all rows of its warps in registers, the CTA's row groups join theirs in
// shared memory, and a second small kernel adds the CTAs' partials in a fixed
// order, so the result is the same in every run.  All arithmetic is fp32; 16-bit
// types are rounded once, at the store.
//
// Widths that are no multiple of the vector (4 elements of an fp32 row, 8 of a
// 16-bit one) begin rows at any of V places in a vector.  The rows of one group
// of warps are V (or a multiple) apart, so that they all begin at the same place
// and a thread's vectors stay aligned and its columns the same; only the first and
// last vector of a row is stored by elements.  A copy takes the 16-byte units that
// hold the row.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <cstdio>
#include <initializer_list>
#include <utility>

#include "cimekv.h"
#include "device_wait.cuh"
#include <nvtx3/nvToolsExt.h>

int cimekv_internal_begin_call();
int cimekv_internal_no_pending_error();
void cimekv_internal_set_error(const char* msg);

namespace {

struct NvtxRange {
    explicit NvtxRange(const char* name) { nvtxRangePushA(name); }
    ~NvtxRange() { nvtxRangePop(); }
};

int fail(int code, const char* msg) {
    cimekv_internal_set_error(msg);
    return code;
}

constexpr int kMaxCols = CIMEKV_LAYER_NORM_MAX_COLS;
constexpr int kReduceLanes = 32;  // partial rows added side by side by one block of the column reduction

__host__ __device__ inline int type_bytes(int type) { return type == CIMEKV_F32 ? 4 : 2; }

// ------------------------------------------------------------- PTX pieces --

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// Copies the 16-byte units that hold `bytes` from `src` (the units before and
// after belong to the same allocation: they hold some of the row).
__device__ __forceinline__ uint32_t units(uintptr_t src, uint32_t bytes) {
    return (((uint32_t)src & 15u) + bytes + 15u) & ~15u;
}
__device__ __forceinline__ void copy_row(uint32_t dst, uintptr_t src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src & ~(uintptr_t)15), "r"(units(src, bytes)), "r"(bar)
                 : "memory");
}

// A row's place in shared memory: room for the units that hold it, and for a
// vector that begins before or ends behind it.
constexpr int kPad = 32;
__host__ __device__ inline uint32_t row_room(int cols, int type) {
    return ((uint32_t)cols * type_bytes(type) + 15 + 2 * kPad + 15) & ~15u;
}

// E vectors of V neighbours of a staged row, vector e at column col0 + e * step, as
// fp32; zeros outside the row.  `at`: shared address of column 0.
template <int V, int E>
__device__ __forceinline__ void read_row(float (&v)[E][V], uint32_t at, int type, int col0, int step, int cols) {
    if (type == CIMEKV_F32) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int col = col0 + e * step;
            uint32_t w[V];
#pragma unroll
            for (int i = 0; i < V; ++i) w[i] = 0u;
            if (col < cols) {
                if constexpr (V == 1) {
                    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(at + col * 4) : "memory");
                } else {
#pragma unroll
                    for (int i = 0; i < V; i += 4)
                        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                     : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3])
                                     : "r"(at + (col + i) * 4)
                                     : "memory");
                }
            }
            if (V > 1 && (col < 0 || col + V > cols)) {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if ((unsigned)(col + i) >= (unsigned)cols) w[i] = 0u;
            }
#pragma unroll
            for (int i = 0; i < V; ++i) v[e][i] = __uint_as_float(w[i]);
        }
        return;
    }
    constexpr int kWords = (V + 1) / 2;
    uint32_t w[E][kWords];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int col = col0 + e * step;
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[e][i] = 0u;
        if (col < cols) {
            const uint32_t from = at + col * 2;
            if constexpr (V == 1) {
                unsigned short h;
                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(from) : "memory");
                w[e][0] = h;
            } else if constexpr (V == 4) {
                asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[e][0]), "=r"(w[e][1]) : "r"(from) : "memory");
            } else {
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(w[e][0]), "=r"(w[e][1]), "=r"(w[e][2]), "=r"(w[e][3])
                             : "r"(from)
                             : "memory");
            }
        }
        if (V > 1 && (col < 0 || col + V > cols)) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if ((unsigned)(col + i) >= (unsigned)cols) w[e][i / 2] &= i % 2 ? 0x0000ffffu : 0xffff0000u;
        }
    }
    if (type == CIMEKV_BF16) {
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int i = 0; i < V; ++i)
                v[e][i] = __uint_as_float(i % 2 ? w[e][i / 2] & 0xffff0000u : w[e][i / 2] << 16);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e][i / 2]));
                v[e][i] = f.x;
                if (i + 1 < V) v[e][i + 1 < V ? i + 1 : i] = f.y;
            }
    }
}

template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if (kBf16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}

template <int V, int E, bool kBf16>
__device__ __forceinline__ void store_row16(const float (&v)[E][V], unsigned short* row, int col0, int step, int cols) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int col = col0 + e * step;
        unsigned short* p = row + col;
        uint32_t w[(V + 1) / 2];
#pragma unroll
        for (int i = 0; i < V; i += 2) w[i / 2] = pack2<kBf16>(v[e][i], i + 1 < V ? v[e][i + 1 < V ? i + 1 : i] : 0.0f);
        if (col >= 0 && col + V <= cols) {
            if constexpr (V == 1) *p = (unsigned short)w[0];
            else if constexpr (V == 4) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
            else *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        } else if (V > 1 && col < cols) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if ((unsigned)(col + i) < (unsigned)cols) p[i] = (unsigned short)(w[i / 2] >> (16 * (i % 2)));
        }
    }
}

// Rounds to `type` and stores.
template <int V, int E>
__device__ __forceinline__ void store_row(const float (&v)[E][V], void* base, int type, int col0, int step, int cols) {
    if (type == CIMEKV_F32) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int col = col0 + e * step;
            float* p = static_cast<float*>(base) + col;
            if (col >= 0 && col + V <= cols) {
                if constexpr (V == 1) {
                    *p = v[e][0];
                } else {
#pragma unroll
                    for (int i = 0; i < V; i += 4)
                        *reinterpret_cast<float4*>(p + i) = make_float4(v[e][i], v[e][i + 1], v[e][i + 2], v[e][i + 3]);
                }
            } else if (V > 1 && col < cols) {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if ((unsigned)(col + i) < (unsigned)cols) p[i] = v[e][i];
            }
        }
    } else if (type == CIMEKV_BF16) {
        store_row16<V, E, true>(v, static_cast<unsigned short*>(base), col0, step, cols);
    } else {
        store_row16<V, E, false>(v, static_cast<unsigned short*>(base), col0, step, cols);
    }
}

// Values as they are after rounding to `type`.
template <int V, int E>
__device__ __forceinline__ void round_row(float (&v)[E][V], int type) {
    if (type == CIMEKV_BF16) {
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int i = 0; i < V; ++i) v[e][i] = __bfloat162float(__float2bfloat16_rn(v[e][i]));
    } else if (type == CIMEKV_F16) {
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int i = 0; i < V; ++i) v[e][i] = __half2float(__float2half_rn(v[e][i]));
    }
}

// Per-column values in registers, for all rows of a thread.
template <int V, int E>
__device__ __forceinline__ void load_columns(float (&v)[E][V], const void* p, int type, float absent, int col0, int stride,
                                             int cols) {
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = col0 + e * stride + i;
            v[e][i] = absent;
            if (p && (unsigned)c < (unsigned)cols) {
                if (type == CIMEKV_F32) v[e][i] = __ldg(static_cast<const float*>(p) + c);
                else if (type == CIMEKV_BF16)
                    v[e][i] = __uint_as_float((uint32_t)__ldg(static_cast<const unsigned short*>(p) + c) << 16);
                else v[e][i] = __half2float(__ushort_as_half(__ldg(static_cast<const unsigned short*>(p) + c)));
            }
        }
}

// Two fp32 operations in one instruction (the same roundings as one by one); both
// directions issue at 60 % without, and most of what they issue is this.
struct Pair {
    float x, y;
};
__device__ __forceinline__ Pair both(float v) { return {v, v}; }
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\t"
        "mov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 d, a, b;\n\t"
        "mov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
// Elements 2 k and 2 k + 1 of a thread (the number of its elements is even).
template <int V, int E>
__device__ __forceinline__ Pair get2(const float (&v)[E][V], int k) {
    return {v[2 * k / V][2 * k % V], v[(2 * k + 1) / V][(2 * k + 1) % V]};
}
template <int V, int E>
__device__ __forceinline__ void set2(float (&v)[E][V], int k, Pair p) {
    v[2 * k / V][2 * k % V] = p.x;
    v[(2 * k + 1) / V][(2 * k + 1) % V] = p.y;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

constexpr int kMaxWarps = 16;
// Rows side by side in a CTA of eight warps (sixteen for the widest rows).
__host__ __device__ constexpr int cta_warps(int W) { return W == 16 ? 16 : 8; }
__host__ __device__ constexpr int cta_rows(int W) { return cta_warps(W) / W; }
__host__ __device__ constexpr int cta_threads(int W) { return cta_warps(W) * 32; }

// CTAs kept resident on an SM: three in the forward where a thread's elements leave
// the registers for it (25.0 -> 22.3 us at 50,432 x 384 fp16, but with 16 elements
// and spilled registers 90 -> 152 us at 16,384 x 4,096), two in the backward
// (three: 40 -> 58 us), one of the widest rows.
__host__ __device__ constexpr int ctas_per_sm(int elements, int W, bool forward) {
    return W == 16 ? 1 : forward && elements <= 12 ? 3 : 2;
}

// Sum over the W warps of a row, the same bits in every thread.  `slot` alternates
// between two buffers, so one barrier of the row's warps is enough: a buffer is
// written again only after the barrier of the sum in between.
template <int W, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*buf)[kMaxWarps][2], int& slot) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
    if constexpr (W > 1) {
        const int warp = threadIdx.x >> 5, group = warp / W;
        if ((threadIdx.x & 31) == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) buf[slot][warp][i] = v[i];
        }
        asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(W * 32) : "memory");
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < W; ++w) s += buf[slot][group * W + w][i];
            v[i] = s;
        }
        slot ^= 1;
    }
}

struct NormParams {
    const void* x;  // forward: x; backward: h
    const void* d;
    const void* dy;
    const void* dh;
    const void* w;
    const void* b;
    void* y;
    void* h;
    void* dx;
    void* dd;
    float* mean;
    float* rstd;
    float* part;
    unsigned* lost;  // marked when a wait has run out
    long long rows, x_stride, d_stride, dy_stride, dh_stride;
    int cols, x_type, d_type, w_type, y_type;
    int stages;  // rows under way per row group
    int places;  // row r begins r * places mod V elements into a vector (the strides mod V)
    float eps;
};

__device__ __forceinline__ void* row_of(void* p, int type, long long row, long long stride) {
    return static_cast<char*>(p) + row * stride * type_bytes(type);
}

constexpr int kMaxStages = 4;

// The rows of one row group on their way through shared memory: up to three
// tensors a row.  One thread of the group copies, all read.
template <int W, int N>
struct Ring {
    uintptr_t next[N];          // address of the row to copy next
    long long step[N];          // bytes from one of the group's rows to the next
    uint32_t low[N];            // low bits of the current row's address
    uint32_t bytes[N], room[N], memory, at_stage, bars, stage_bytes;
    int stages, stage, phase, lost;
    bool ok;

    __device__ __forceinline__ void tensor(int k, const void* base, int type, long long stride, long long row, long long rows_apart,
                                           int cols) {
        const int size = type_bytes(type);
        next[k] = (uintptr_t)base + row * stride * size;
        low[k] = (uint32_t)next[k];
        step[k] = rows_apart * stride * size;
        bytes[k] = (uint32_t)cols * size;
        room[k] = row_room(cols, type);
    }
    // `memory_`: of the CTA; `bars_`: the group's kMaxStages barriers.  All threads of
    // the CTA, after its tensors.
    __device__ __forceinline__ void open(uint32_t memory_, uint32_t bars_, int stages_) {
        stages = stages_;
        stage_bytes = 0;
#pragma unroll
        for (int k = 0; k < N; ++k) stage_bytes += room[k];
        at_stage = memory = memory_ + threadIdx.x / (W * 32) * stages * stage_bytes;
        bars = bars_;
        stage = phase = lost = 0;
        ok = true;
        if (threadIdx.x % (W * 32) == 0) {
            for (int s = 0; s < kMaxStages; ++s)
                asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bars + 8 * s) : "memory");
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncthreads();
    }
    // The group's next row into `place`, by the copying thread.
    __device__ __forceinline__ void copy(int place) {
        uint32_t total = 0;
#pragma unroll
        for (int k = 0; k < N; ++k) total += units(next[k], bytes[k]);
        const uint32_t bar = bars + 8 * place;
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(total) : "memory");
        uint32_t dst = memory + place * stage_bytes + kPad;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            copy_row(dst, next[k], bytes[k], bar);
            dst += room[k];
            next[k] += step[k];
        }
    }
    // The next row of the group is in shared memory.  After a wait that ran out
    // no row is copied any more; those under way are still waited for.
    __device__ __forceinline__ void wait() {
        if (lost == stages) return;
        ok = mbar_wait(bars + 8 * stage, phase) && ok;
        if (!ok) ++lost;
    }
    // Shared address of column 0 of tensor k of the current row.
    __device__ __forceinline__ uint32_t at(int k) const {
        uint32_t a = at_stage + kPad + (low[k] & 15u);
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < k) a += room[i];
        return a;
    }
    // After all threads of the group have read the current row (and met): its
    // place takes another one, if there is one.
    __device__ __forceinline__ void take(bool more) {
        if (threadIdx.x % (W * 32) == 0 && more && ok) copy(stage);
#pragma unroll
        for (int k = 0; k < N; ++k) low[k] += (uint32_t)step[k];
        at_stage += stage_bytes;
        if (++stage == stages) {
            stage = 0;
            at_stage = memory;
            phase ^= 1;
        }
    }
};

// s / n to the last bit or so, by a reciprocal taken once.
__device__ __forceinline__ float divide(float s, float n, float inv) {
    const float q = s * inv;
    return fmaf(fmaf(-q, n, s), inv, q);
}

// All threads of a row's warps meet.
template <int W>
__device__ __forceinline__ void row_sync() {
    if constexpr (W == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"((int)threadIdx.x / (W * 32) + 1), "n"(W * 32) : "memory");
}

// Measured (copy bandwidth 6.5 TB/s): 16,384 x 4,096 bf16 with a branch in 92 us, 5.9
// TB/s; 32,736 x 768 fp32 with a bf16 branch in 55 us, 5.5 TB/s; 4,099 x 1,537 bf16 with a
// branch (inside L2) in 18 us, where the instructions count: 69 % of the issue slots at
// 50,432 x 384 fp16 (22 us), two or three warps of a scheduler waiting for a row's sums.
template <int V, int E, int W, bool kDelta>
__global__ void __launch_bounds__(cta_threads(W), ctas_per_sm(V * E, W, true)) norm_fwd_kernel(NormParams p) {
    constexpr int T = W * 32, kStep = T * V, N = kDelta ? 2 : 1;
    extern __shared__ __align__(16) uint8_t memory[];
    __shared__ __align__(8) uint64_t bars[cta_rows(W)][kMaxStages];
    __shared__ float red[2][kMaxWarps][2];
    int slot = 0;
    const int t = threadIdx.x % T, group = threadIdx.x / T;
    long long row = (long long)blockIdx.x * cta_rows(W) + group;
    const long long step = (long long)gridDim.x * cta_rows(W);
    const int col0 = t * V - (int)((unsigned)row * (unsigned)p.places % V);
    const float n = (float)p.cols, inv = 1.0f / n;
    Ring<W, N> ring;
    ring.tensor(0, p.x, p.x_type, p.x_stride, row, step, p.cols);
    if constexpr (kDelta) ring.tensor(1, p.d, p.d_type, p.d_stride, row, step, p.cols);
    ring.open(smem_addr(memory), smem_addr(bars[group]), p.stages);
    if (row >= p.rows) return;  // whole groups of warps
    if (t == 0)
        for (int s = 0; s < p.stages && row + s * step < p.rows; ++s) ring.copy(s);
    float w[E][V], b[E][V];
    load_columns(w, p.w, p.w_type, 1.0f, col0, kStep, p.cols);
    load_columns(b, p.b, p.w_type, 0.0f, col0, kStep, p.cols);
    for (; row < p.rows; row += step) {
        float h[E][V];
        ring.wait();
        read_row<V, E>(h, ring.at(0), p.x_type, col0, kStep, p.cols);
        if constexpr (kDelta) {
            float d[E][V];
            read_row<V, E>(d, ring.at(1), p.d_type, col0, kStep, p.cols);
#pragma unroll
            for (int k = 0; k < E * V / 2; ++k) set2(h, k, add2(get2(h, k), get2(d, k)));
            store_row<V, E>(h, row_of(p.h, p.x_type, row, p.cols), p.x_type, col0, kStep, p.cols);
            // y is the norm of the sum as it is held (and as the backward reads it)
            round_row<V, E>(h, p.x_type);
        }
        Pair sum = both(0.0f);
#pragma unroll
        for (int k = 0; k < E * V / 2; ++k) sum = add2(sum, get2(h, k));
        float s[1] = {sum.x + sum.y};
        row_sum<W, 1>(s, red, slot);
        if (W == 1) __syncwarp();
        ring.take(row + p.stages * step < p.rows);  // the sum was taken by all: all have read
        const float mean = ring.ok ? divide(s[0], n, inv) : __int_as_float(0x7fffffff);  // a lost copy shows as NaN
        const Pair minus = both(-mean);
#pragma unroll
        for (int k = 0; k < E * V / 2; ++k) set2(h, k, add2(get2(h, k), minus));
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int col = col0 + e * kStep;
            if (col < 0 || col + V > p.cols) {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if ((unsigned)(col + i) >= (unsigned)p.cols) h[e][i] = 0.0f;
            }
        }
        Pair squares = both(0.0f);
#pragma unroll
        for (int k = 0; k < E * V / 2; ++k) squares = fma2(get2(h, k), get2(h, k), squares);
        float q[1] = {squares.x + squares.y};
        row_sum<W, 1>(q, red, slot);
        const float rstd = rsqrtf(divide(q[0], n, inv) + p.eps);
        if (t == 0 && p.mean) {
            p.mean[row] = mean;
            p.rstd[row] = rstd;
        }
#pragma unroll
        for (int k = 0; k < E * V / 2; ++k)
            set2(h, k, fma2(mul2(get2(h, k), both(rstd)), get2(w, k), get2(b, k)));
        store_row<V, E>(h, row_of(p.y, p.y_type, row, p.cols), p.y_type, col0, kStep, p.cols);
    }
    if (!ring.ok) mark_lost(p.lost);
}

// kSum: the sum's own gradient dh is added to dx.  p.part: the CTA's column sums
// [gridDim][2][cols] (dw, db), or null when no weight gradient is wanted.
// Measured: 16,384 x 4,096 bf16 with dh in 105 us, 5.1 TB/s; 32,736 x 768 fp32, bf16
// branch, in 74 to 78 us, 5.2 TB/s and more; 50,432 x 384 fp16, fp32 dy, in 40 us, 3.9 TB/s: rows this
// short pay for their two sums (48 % of the issue slots, the rest is their latency).
template <int V, int E, int W, bool kSum>
__global__ void __launch_bounds__(cta_threads(W), ctas_per_sm(V * E, W, false)) norm_bwd_kernel(NormParams p) {
    constexpr int T = W * 32, kStep = T * V, N = kSum ? 3 : 2;
    extern __shared__ __align__(16) uint8_t memory[];
    __shared__ __align__(8) uint64_t bars[cta_rows(W)][kMaxStages];
    __shared__ float red[2][kMaxWarps][2];
    int slot = 0;
    const int t = threadIdx.x % T, group = threadIdx.x / T;
    long long row = (long long)blockIdx.x * cta_rows(W) + group;
    const long long step = (long long)gridDim.x * cta_rows(W);
    const int col0 = t * V - (int)((unsigned)row * (unsigned)p.places % V);
    const float n = (float)p.cols, inv = 1.0f / n;
    Ring<W, N> ring;
    ring.tensor(0, p.x, p.x_type, p.x_stride, row, step, p.cols);
    ring.tensor(1, p.dy, p.y_type, p.dy_stride, row, step, p.cols);
    if constexpr (kSum) ring.tensor(2, p.dh, p.x_type, p.dh_stride, row, step, p.cols);
    ring.open(smem_addr(memory), smem_addr(bars[group]), p.stages);
    float dw[E][V] = {}, db[E][V] = {};
    if (row < p.rows) {
        if (t == 0)
            for (int s = 0; s < p.stages && row + s * step < p.rows; ++s) ring.copy(s);
        float w[E][V];
        load_columns(w, p.w, p.w_type, 1.0f, col0, kStep, p.cols);
        float next_mean = __ldg(p.mean + row), next_rstd = __ldg(p.rstd + row);
        for (; row < p.rows; row += step) {
            const float mean = next_mean, rstd = next_rstd;
            if (row + step < p.rows) {
                next_mean = __ldg(p.mean + row + step);
                next_rstd = __ldg(p.rstd + row + step);
            }
            float u[E][V], g[E][V];
            ring.wait();
            read_row<V, E>(u, ring.at(0), p.x_type, col0, kStep, p.cols);
            read_row<V, E>(g, ring.at(1), p.y_type, col0, kStep, p.cols);
            const Pair minus = both(-mean), unit = both(rstd);
            Pair s0 = both(0.0f), s1 = both(0.0f);
#pragma unroll
            for (int k = 0; k < E * V / 2; ++k) {  // outside the row g is zero, and u only meets g
                const Pair v = mul2(add2(get2(u, k), minus), unit), y = get2(g, k);
                set2(u, k, v);
                set2(dw, k, fma2(y, v, get2(dw, k)));
                set2(db, k, add2(y, get2(db, k)));
                const Pair z = mul2(y, get2(w, k));
                set2(g, k, z);
                s0 = add2(z, s0);
                s1 = fma2(z, v, s1);
            }
            float s[2] = {s0.x + s0.y, s1.x + s1.y};
            row_sum<W, 2>(s, red, slot);
            const float scale = ring.ok ? rstd : __int_as_float(0x7fffffff);  // a lost copy shows as NaN
            const Pair c1 = both(-scale * divide(s[0], n, inv)), c2 = both(-scale * divide(s[1], n, inv));
#pragma unroll
            for (int k = 0; k < E * V / 2; ++k)
                set2(g, k, fma2(both(scale), get2(g, k), fma2(c2, get2(u, k), c1)));
            if constexpr (kSum) {
                read_row<V, E>(u, ring.at(2), p.x_type, col0, kStep, p.cols);
#pragma unroll
                for (int k = 0; k < E * V / 2; ++k) set2(g, k, add2(get2(g, k), get2(u, k)));
            }
            if (kSum || W == 1) row_sync<W>();
            ring.take(row + p.stages * step < p.rows);
            if (p.dx) store_row<V, E>(g, row_of(p.dx, p.x_type, row, p.cols), p.x_type, col0, kStep, p.cols);
            if (p.dd) store_row<V, E>(g, row_of(p.dd, p.d_type, row, p.cols), p.d_type, col0, kStep, p.cols);
        }
        if (!ring.ok) {
            dw[0][0] = db[0][0] = __int_as_float(0x7fffffff);
            mark_lost(p.lost);
        }
    }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (!p.part) return;
    // [2][cols] where row groups share a CTA, over the rows' places once all are taken
    float* join = reinterpret_cast<float*>(memory);
    float* out = p.part + (long long)blockIdx.x * 2 * p.cols;
    float* to = cta_rows(W) > 1 ? join : out;
    __syncthreads();
    for (int g = 0; g < cta_rows(W); ++g) {  // one row group after the other: a fixed order
        if (group == g) {
#pragma unroll
            for (int e = 0; e < E; ++e)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const int c = col0 + e * kStep + i;
                    if ((unsigned)c < (unsigned)p.cols) {
                        to[c] = g ? to[c] + dw[e][i] : dw[e][i];
                        to[p.cols + c] = g ? to[p.cols + c] + db[e][i] : db[e][i];
                    }
                }
        }
        if (cta_rows(W) > 1) __syncthreads();
    }
    if (cta_rows(W) > 1)
        for (int c = threadIdx.x; c < 2 * p.cols; c += cta_threads(W)) out[c] = join[c];
}

// dw / db (blockIdx.y) of 32 columns: kReduceLanes partial rows side by side,
// then a fixed tree over them.  2 to 3 us, part of it under the end of the rows' kernel.
__global__ void __launch_bounds__(32 * kReduceLanes) norm_cols_kernel(const float* part, int nparts, int cols, void* dw,
                                                                       void* db, int type) {
    __shared__ float s[kReduceLanes][33];
    void* out = blockIdx.y ? db : dw;
    if (!out) return;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int c = blockIdx.x * 32 + threadIdx.x;
    float v = 0.0f;
    if (c < cols) {
        const float* src = part + (long long)blockIdx.y * cols + c;
#pragma unroll 8
        for (int r = threadIdx.y; r < nparts; r += kReduceLanes) v += src[(long long)r * 2 * cols];
    }
    s[threadIdx.y][threadIdx.x] = v;
    __syncthreads();
    v = warp_sum(s[threadIdx.x][threadIdx.y]);  // warp y: the lanes' sums of column y
    const int col = blockIdx.x * 32 + threadIdx.y;
    if (threadIdx.x == 0 && col < cols) {
        if (type == CIMEKV_F32) static_cast<float*>(out)[col] = v;
        else if (type == CIMEKV_BF16) static_cast<__nv_bfloat16*>(out)[col] = __float2bfloat16_rn(v);
        else static_cast<__half*>(out)[col] = __float2half_rn(v);
    }
}

// ------------------------------------------------------------------ host ----

struct Shape {
    int v, e, w;
    constexpr int capacity() const { return v * e * w * 32; }
};

// Layouts of a row by width, for vectors of 4 (fp32 rows), of 8 (16-bit rows) and
// single elements (strides or addresses that no vector fits): the first that
// holds the row is taken.  Measured over 64 Mi elements, forward and backward in TB/s:
//                fp32         bf16         bf16 by single elements
//      384    5.7   6.0    3.8   4.2    1.1   1.2
//    1,024    5.9   5.2    4.5   3.3    2.7   3.1
//    1,280    5.1   4.2    2.9   2.4    1.1   1.3    (a quarter and more of the threads idle between layouts)
//    1,536    6.0   4.4    3.4   2.8    1.2   1.5
//    4,096    5.8   5.8    4.2   4.5    2.7   3.6
//    5,120    4.3   5.1    1.3   1.5    1.1   0.8    (16-bit: four CTAs take a second turn, see grid_size)
//    8,192    5.7   6.2    2.0   2.3    1.6   1.1
//   16,384    5.8   3.4    2.0   1.3    2.4   1.8    (32 elements a thread)
// The backward has 128 registers a thread: with 16 elements in it it spills up to 140 bytes, with 32 about 1 KB.
constexpr Shape kShapes[] = {{4, 1, 1}, {4, 2, 1}, {4, 3, 1}, {4, 4, 1}, {4, 3, 2}, {4, 4, 2}, {4, 4, 4}, {4, 4, 8},
                             {4, 4, 16}, {4, 8, 16},
                             {8, 1, 1}, {8, 2, 1}, {8, 2, 2}, {8, 2, 4}, {8, 2, 8}, {8, 2, 16}, {8, 4, 16},
                             {1, 8, 1}, {1, 8, 4}, {1, 16, 8}, {1, 32, 16}};
constexpr int kNumShapes = sizeof(kShapes) / sizeof(kShapes[0]);

// inside: rows begin inside a vector, by their strides whatever their width: room for one
// vector more.
int pick_shape(int cols, int v, bool inside) {
    for (int i = 0; i < kNumShapes; ++i)
        if (kShapes[i].v == v && kShapes[i].capacity() >= cols + (inside || cols % v ? v - 1 : 0)) return i;
    return -1;
}

using Kernel = void (*)(NormParams);
struct Kernels {
    Kernel fwd[2], bwd[2];  // without and with a branch / a gradient of the sum
};
template <int I>
constexpr Kernels kernels_of() {
    constexpr Shape s = kShapes[I];
    return {{norm_fwd_kernel<s.v, s.e, s.w, false>, norm_fwd_kernel<s.v, s.e, s.w, true>},
            {norm_bwd_kernel<s.v, s.e, s.w, false>, norm_bwd_kernel<s.v, s.e, s.w, true>}};
}
template <int... I>
const Kernels& kernels(int i, std::integer_sequence<int, I...>) {
    static const Kernels table[] = {kernels_of<I>()...};
    return table[i];
}
const Kernels& kernels(int i) { return kernels(i, std::make_integer_sequence<int, kNumShapes>()); }

// Rows under way per row group: as many as fit a CTA's share of 200 KB of shared
// memory, at most four.
int ring_stages(const Shape& s, size_t row_bytes, bool forward) {
    const size_t share = (200 << 10) / ctas_per_sm(s.v * s.e, s.w, forward);
    const size_t n = share / (row_bytes * cta_rows(s.w));
    return n > kMaxStages ? kMaxStages : n < 1 ? 1 : (int)n;
}

int sm_count(int* sms) {
    int dev;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        return fail(CIMEKV_ECUDA, "cannot read the device's SM count");
    return CIMEKV_OK;
}

// CTAs of a launch: what is resident at once; a multiple of V, so that a group's rows
// all begin at the same place of a vector.  (One CTA an SM and V = 8 make it 152 for 148 places, which
// costs the widest 16-bit rows a second turn.)
long long grid_size(long long rows, const Shape& s, int sms, bool forward) {
    const long long need = (rows + cta_rows(s.w) - 1) / cta_rows(s.w);
    const long long most = (long long)sms * ctas_per_sm(s.v * s.e, s.w, forward);
    return ((need < most ? need : most) + s.v - 1) / s.v * s.v;
}

bool valid_type(int t) { return t == CIMEKV_F32 || t == CIMEKV_BF16 || t == CIMEKV_F16; }

// One tensor of a call: address, type, row stride.
struct Tensor {
    const void* p;
    int type;
    long long stride;
};

// Whether vectors of v elements fit: every address is a multiple, and all rows
// begin at the same places.  places: how far a row's beginning moves in a vector
// from row to row.
bool vectors_fit(int v, std::initializer_list<Tensor> ts, int* places) {
    *places = -1;
    for (const Tensor& t : ts) {
        if (!t.p) continue;
        const int here = (int)(t.stride % v);
        if ((uintptr_t)t.p % ((size_t)v * type_bytes(t.type)) != 0 || (*places >= 0 && *places != here)) return false;
        *places = here;
    }
    if (*places < 0) *places = 0;
    return true;
}

// The layout for a call's tensors.  16-bit rows take vectors of eight, or of four
// where those leave fewer threads idle (384 columns: 384 places against 512).
int layout_of(int x_type, int cols, std::initializer_list<Tensor> ts, int* places) {
    const bool fours = vectors_fit(4, ts, places);
    const int four = fours ? pick_shape(cols, 4, *places != 0) : -1;
    int places8;
    if (x_type != CIMEKV_F32 && vectors_fit(8, ts, &places8)) {
        const int eight = pick_shape(cols, 8, places8 != 0);
        if (eight >= 0 && (four < 0 || kShapes[eight].capacity() <= kShapes[four].capacity())) {
            *places = places8;
            return eight;
        }
    }
    if (four >= 0) return four;
    *places = 0;
    return pick_shape(cols, 1, false);
}

// Lets kernel number `id` use as much shared memory as its layout may ask for, once
// per device (the attribute stays).
int allow_smem(const void* kernel, int id, size_t bytes) {
    static std::atomic<uint64_t> done[4 * kNumShapes];
    if (bytes <= (47 << 10)) return CIMEKV_OK;  // 48 KB need no leave, the kernels' own variables (384 bytes) among them
    int dev;
    if (cudaGetDevice(&dev) != cudaSuccess) return fail(CIMEKV_ECUDA, "no current device");
    if (dev < 64 && (done[id].load(std::memory_order_acquire) >> dev & 1)) return CIMEKV_OK;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 << 10);
    if (e != cudaSuccess) return fail(CIMEKV_ECUDA, cudaGetErrorString(e));
    if (dev < 64) done[id].fetch_or(1ull << dev, std::memory_order_release);
    return CIMEKV_OK;
}

int check_sizes(long long rows, int cols) {
    if (rows < 0) return fail(CIMEKV_EINVAL_SHAPE, "negative number of rows");
    if (cols < 1 || cols > kMaxCols) {
        char msg[128];
        snprintf(msg, sizeof(msg), "layer norm takes 1 to %d columns, got %d", kMaxCols, cols);
        return fail(CIMEKV_EINVAL_SHAPE, msg);
    }
    return CIMEKV_OK;
}

int launched(const char* what) {
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) return CIMEKV_OK;
    char msg[256];
    snprintf(msg, sizeof(msg), "%s: %s", what, cudaGetErrorString(e));
    return fail(CIMEKV_ECUDA, msg);
}

}  // namespace

extern "C" int cimekv_layer_norm_forward(const void* x, int x_type, long long x_stride, const void* delta,
                                         int delta_type, long long delta_stride, const void* weight, const void* bias,
                                         int w_type, long long rows, int cols, float eps, void* h, void* y, int y_type,
                                         float* mean, float* rstd, void* stream) {
    NvtxRange nvtx_range("cimekv_layer_norm_forward");
    int rc = cimekv_internal_begin_call();
    if (rc || (rc = check_sizes(rows, cols))) return rc;
    if (!valid_type(x_type) || !valid_type(y_type) || !valid_type(w_type) || (delta && !valid_type(delta_type)))
        return fail(CIMEKV_EINVAL_SHAPE, "unknown element type");
    if (!(eps >= 0.0f)) return fail(CIMEKV_EINVAL_SHAPE, "eps must be >= 0");
    if (rows == 0) return CIMEKV_OK;
    if (!x || !y || (delta != nullptr) != (h != nullptr) || (mean != nullptr) != (rstd != nullptr))
        return fail(CIMEKV_EINVAL_SHAPE, "null pointer");
    if (x_stride < 0 || delta_stride < 0) return fail(CIMEKV_EINVAL_SHAPE, "negative stride");
    int places, sms;
    const int i = layout_of(x_type, cols, {{x, x_type, x_stride}, {delta, delta_type, delta_stride}, {h, x_type, cols},
                                           {y, y_type, cols}}, &places);
    if ((rc = sm_count(&sms))) return rc;
    NormParams p = {};
    p.x = x;
    p.d = delta;
    p.w = weight;
    p.b = bias;
    p.h = h;
    p.y = y;
    p.mean = mean;
    p.rstd = rstd;
    p.rows = rows;
    p.cols = cols;
    p.x_stride = x_stride;
    p.d_stride = delta_stride;
    p.x_type = x_type;
    p.d_type = delta_type;
    p.w_type = w_type;
    p.y_type = y_type;
    p.places = places;
    p.eps = eps;
    if ((rc = cimekv_internal_no_pending_error()) || (rc = cimekv_internal_wait_word(CIMEKV_WAIT_NORM, &p.lost))) return rc;
    const size_t row_bytes = row_room(cols, x_type) + (delta ? row_room(cols, delta_type) : 0);
    p.stages = ring_stages(kShapes[i], row_bytes, true);
    const Kernel kernel = kernels(i).fwd[delta != nullptr];
    const size_t smem = row_bytes * p.stages * cta_rows(kShapes[i].w);
    if ((rc = allow_smem((const void*)kernel, 4 * i + (delta != nullptr), smem))) return rc;
    kernel<<<(unsigned)grid_size(rows, kShapes[i], sms, true), cta_threads(kShapes[i].w), smem, (cudaStream_t)stream>>>(p);
    return launched("norm_fwd_kernel");
}

// The widest grid any layout takes, so that the size does not depend on
// addresses (which decide between the vector and the scalar layout).
extern "C" size_t cimekv_layer_norm_workspace_bytes(long long rows, int cols) {
    if (rows <= 0 || cols < 1 || cols > kMaxCols) return 0;
    int sms;
    if (sm_count(&sms)) return 0;
    long long most = 0;
    for (const int v : {1, 4, 8}) {
        for (const bool inside : {false, true}) {
            const int i = pick_shape(cols, v, inside);
            const long long g = i < 0 ? 0 : grid_size(rows, kShapes[i], sms, false);
            if (g > most) most = g;
        }
    }
    return (size_t)most * 2 * (size_t)cols * sizeof(float);
}

extern "C" int cimekv_layer_norm_backward(const void* dy, int y_type, long long dy_stride, const void* dh,
                                          long long dh_stride, const void* h, int x_type, long long h_stride,
                                          const void* weight, int w_type, const float* mean, const float* rstd,
                                          long long rows, int cols, void* dx, void* ddelta, int delta_type, void* dw,
                                          void* db, void* workspace, size_t workspace_bytes, void* stream) {
    NvtxRange nvtx_range("cimekv_layer_norm_backward");
    int rc = cimekv_internal_begin_call();
    if (rc || (rc = check_sizes(rows, cols))) return rc;
    if (!valid_type(x_type) || !valid_type(y_type) || !valid_type(w_type) || (ddelta && !valid_type(delta_type)))
        return fail(CIMEKV_EINVAL_SHAPE, "unknown element type");
    const bool want_w = dw || db;
    if (!dx && !ddelta && !want_w) return CIMEKV_OK;
    if (rows > 0 && (!dy || !h || !mean || !rstd)) return fail(CIMEKV_EINVAL_SHAPE, "null pointer");
    if (h_stride < 0 || dy_stride < 0 || dh_stride < 0) return fail(CIMEKV_EINVAL_SHAPE, "negative stride");
    cudaStream_t s = (cudaStream_t)stream;
    int nparts = 0;
    if (rows > 0) {
        int places, sms;
        const int i = layout_of(x_type, cols, {{h, x_type, h_stride}, {dy, y_type, dy_stride}, {dh, x_type, dh_stride},
                                               {dx, x_type, cols}, {ddelta, delta_type, cols}}, &places);
        if ((rc = sm_count(&sms))) return rc;
        const long long grid = grid_size(rows, kShapes[i], sms, false);
        if (want_w) {
            if (!workspace || workspace_bytes < (size_t)grid * 2 * cols * sizeof(float))
                return fail(CIMEKV_EWORKSPACE, "layer norm backward workspace too small");
            if ((uintptr_t)workspace % 16) return fail(CIMEKV_EINVAL_SHAPE, "workspace must be 16-byte aligned");
        }
        NormParams p = {};
        p.x = h;
        p.dy = dy;
        p.dh = dh;
        p.w = weight;
        p.dx = dx;
        p.dd = ddelta;
        p.mean = const_cast<float*>(mean);
        p.rstd = const_cast<float*>(rstd);
        p.part = want_w ? static_cast<float*>(workspace) : nullptr;
        p.rows = rows;
        p.cols = cols;
        p.x_stride = h_stride;
        p.dy_stride = dy_stride;
        p.dh_stride = dh_stride;
        p.x_type = x_type;
        p.d_type = delta_type;
        p.w_type = w_type;
        p.y_type = y_type;
        p.places = places;
        const size_t row_bytes = row_room(cols, y_type) + (dh ? 2 : 1) * (size_t)row_room(cols, x_type);
        p.stages = ring_stages(kShapes[i], row_bytes, false);
        const Kernel kernel = kernels(i).bwd[dh != nullptr];
        size_t smem = row_bytes * p.stages * cta_rows(kShapes[i].w);
        if (cta_rows(kShapes[i].w) > 1 && smem < (size_t)2 * cols * sizeof(float)) smem = (size_t)2 * cols * sizeof(float);
        if ((rc = cimekv_internal_no_pending_error()) || (rc = cimekv_internal_wait_word(CIMEKV_WAIT_NORM, &p.lost)) ||
            (rc = allow_smem((const void*)kernel, 4 * i + 2 + (dh != nullptr), smem)))
            return rc;
        kernel<<<(unsigned)grid, cta_threads(kShapes[i].w), smem, s>>>(p);
        if ((rc = launched("norm_bwd_kernel"))) return rc;
        nparts = (int)grid;
    } else if ((rc = cimekv_internal_no_pending_error())) {
        return rc;
    }
    if (!want_w) return CIMEKV_OK;
    // no rows: the sums over none of them are zero
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(cols + 31) / 32, 2);
    cfg.blockDim = dim3(32, kReduceLanes);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // set up while the rows finish
    attr[0].val.programmaticStreamSerializationAllowed = rows > 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, norm_cols_kernel, static_cast<const float*>(workspace), nparts, cols, dw,
                                             db, w_type);
    if (e == cudaSuccess) return CIMEKV_OK;
    (void)cudaGetLastError();
    return fail(CIMEKV_ECUDA, cudaGetErrorString(e));
}
