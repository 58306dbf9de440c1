// layer_norm.cu — layer normalisation and its backward pass, alone and joined
// with the residual sum in front of it.
//
//   h = x + d (rounded to h's type; h = x without a branch d)
//   u = (h - mean(h)) * rstd,  rstd = (var(h) + eps)^-1/2,  y = u w + b
//   dx = rstd (g w - mean(g w) - u mean(g w u)) + dh,  dw = sum_rows g u,  db = sum_rows g
//
// Both directions are bound by HBM: every row is read once into registers, the
// row sums are taken there (mean first, then the centred squares: no
// cancellation for rows far from zero), and the results leave in the same pass.
// A row belongs to one warp up to 1024 columns, to one CTA above.  The weight
// gradients are column sums: each thread keeps the sums of its own columns over
// all rows of its CTA in registers, the CTA's warps join theirs in shared memory,
// and a second small kernel adds the CTAs' partials in a fixed order, so the
// result is the same in every run.  All arithmetic is fp32; 16-bit types are
// rounded once, at the store.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <cstdio>

#include "cimekv.h"
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

// One row's elements of a thread: E groups of V neighbours, groups T*V apart.
template <int V, int E>
struct Row {
    uint32_t raw[E][V];  // fp32 bits; two 16-bit values to a word while raw (V = 4), one in the low half (V = 1)

    // Issues the row's loads; nothing here waits for them.
    __device__ __forceinline__ void load(const void* base, int type, int t, int T, int cols) {
        if (type == CIMEKV_F32) {
            const float* p = static_cast<const float*>(base);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int col = (e * T + t) * V;
                if (col < cols) {
                    if constexpr (V == 4) {
                        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p + col));
                        raw[e][0] = v.x; raw[e][1] = v.y; raw[e][2] = v.z; raw[e][3] = v.w;
                    } else {
                        raw[e][0] = __float_as_uint(__ldg(p + col));
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i) raw[e][i] = 0u;
                }
            }
        } else {
            const unsigned short* p = static_cast<const unsigned short*>(base);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int col = (e * T + t) * V;
                if (col < cols) {
                    if constexpr (V == 4) {
                        const uint2 v = __ldg(reinterpret_cast<const uint2*>(p + col));
                        raw[e][0] = v.x; raw[e][1] = v.y;
                    } else {
                        raw[e][0] = __ldg(p + col);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < (V == 4 ? 2 : 1); ++i) raw[e][i] = 0u;
                }
            }
        }
    }

    // Raw words to fp32 bits, in place.
    __device__ __forceinline__ void widen(int type) {
        if (type == CIMEKV_F32) return;
        if (type == CIMEKV_BF16) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if constexpr (V == 4) {
                    const uint32_t a = raw[e][0], b = raw[e][1];
                    raw[e][0] = a << 16; raw[e][1] = a & 0xffff0000u;
                    raw[e][2] = b << 16; raw[e][3] = b & 0xffff0000u;
                } else {
                    raw[e][0] <<= 16;
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if constexpr (V == 4) {
                    const uint32_t a = raw[e][0], b = raw[e][1];
                    raw[e][0] = half_bits(a); raw[e][1] = half_bits(a >> 16);
                    raw[e][2] = half_bits(b); raw[e][3] = half_bits(b >> 16);
                } else {
                    raw[e][0] = half_bits(raw[e][0]);
                }
            }
        }
    }

    static __device__ __forceinline__ uint32_t half_bits(uint32_t h) {
        return __float_as_uint(__half2float(__ushort_as_half((unsigned short)h)));
    }
    __device__ __forceinline__ float get(int e, int i) const { return __uint_as_float(raw[e][i]); }
    __device__ __forceinline__ void set(int e, int i, float v) { raw[e][i] = __float_as_uint(v); }

    // Rounds to `type` and stores; what the row then holds is not rounded.
    __device__ __forceinline__ void store(void* base, int type, int t, int T, int cols) const {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int col = (e * T + t) * V;
            if (col >= cols) continue;
            if (type == CIMEKV_F32) {
                float* p = static_cast<float*>(base) + col;
                if constexpr (V == 4) *reinterpret_cast<uint4*>(p) = make_uint4(raw[e][0], raw[e][1], raw[e][2], raw[e][3]);
                else *p = get(e, 0);
            } else {
                unsigned short* p = static_cast<unsigned short*>(base) + col;
                unsigned short s[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    s[i] = type == CIMEKV_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(get(e, i)))
                                               : __half_as_ushort(__float2half_rn(get(e, i)));
                }
                if constexpr (V == 4)
                    *reinterpret_cast<uint2*>(p) = make_uint2(s[0] | (uint32_t)s[1] << 16, s[2] | (uint32_t)s[3] << 16);
                else
                    *p = s[0];
            }
        }
    }
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Sum over the W warps of a row (W == 1: the row's own warp), the same bits in
// every thread.  `slot` alternates between two buffers, so one barrier is enough:
// a buffer is written again only after the barrier of the sum in between.
template <int W, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*buf)[W][N], int& slot) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
    if constexpr (W > 1) {
        float(*b)[N] = buf[slot];
        if ((threadIdx.x & 31) == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) b[threadIdx.x >> 5][i] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < W; ++w) s += b[w][i];
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
    long long rows, x_stride, d_stride, dy_stride, dh_stride;
    int cols, x_type, d_type, w_type, y_type;
    float eps;
};

__device__ __forceinline__ const void* row_of(const void* p, int type, long long row, long long stride) {
    return static_cast<const char*>(p) + row * stride * type_bytes(type);
}
__device__ __forceinline__ void* row_of(void* p, int type, long long row, long long stride) {
    return static_cast<char*>(p) + row * stride * type_bytes(type);
}

// Threads of a CTA: one row per CTA above one warp per row, eight rows below.
__host__ __device__ constexpr int cta_threads(int W) { return W == 1 ? 256 : W * 32; }
__host__ __device__ constexpr int cta_rows(int W) { return W == 1 ? 8 : 1; }

template <int V, int E, int W, bool kDelta>
__global__ void __launch_bounds__(cta_threads(W)) norm_fwd_kernel(NormParams p) {
    constexpr int T = W * 32;
    __shared__ float red[2][W][1];
    int slot = 0;
    const int t = W == 1 ? (threadIdx.x & 31) : threadIdx.x;
    const long long first = W == 1 ? (long long)blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x;
    for (long long row = first; row < p.rows; row += (long long)gridDim.x * cta_rows(W)) {
        Row<V, E> h;
        h.load(row_of(p.x, p.x_type, row, p.x_stride), p.x_type, t, T, p.cols);
        if constexpr (kDelta) {
            Row<V, E> d;
            d.load(row_of(p.d, p.d_type, row, p.d_stride), p.d_type, t, T, p.cols);
            h.widen(p.x_type);
            d.widen(p.d_type);
#pragma unroll
            for (int e = 0; e < E; ++e)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    float s = h.get(e, i) + d.get(e, i);
                    // y is the norm of the sum as it is held (and as the backward reads it)
                    if (p.x_type == CIMEKV_BF16) s = __bfloat162float(__float2bfloat16_rn(s));
                    else if (p.x_type == CIMEKV_F16) s = __half2float(__float2half_rn(s));
                    h.set(e, i, s);
                }
            h.store(row_of(p.h, p.x_type, row, p.cols), p.x_type, t, T, p.cols);
        } else {
            h.widen(p.x_type);
        }
        float s[1] = {0.0f};
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int i = 0; i < V; ++i) s[0] += h.get(e, i);
        row_sum<W, 1>(s, red, slot);
        const float mean = s[0] / (float)p.cols;
        float q[1] = {0.0f};
#pragma unroll
        for (int e = 0; e < E; ++e)
            if ((e * T + t) * V < p.cols) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float c = h.get(e, i) - mean;
                    h.set(e, i, c);
                    q[0] = fmaf(c, c, q[0]);
                }
            }
        row_sum<W, 1>(q, red, slot);
        const float rstd = rsqrtf(q[0] / (float)p.cols + p.eps);
        if (t == 0 && p.mean) {
            p.mean[row] = mean;
            p.rstd[row] = rstd;
        }
        Row<V, E> w;
        if (p.w) {
            w.load(p.w, p.w_type, t, T, p.cols);
            w.widen(p.w_type);
        }
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float u = h.get(e, i) * rstd;
                h.set(e, i, p.w ? u * w.get(e, i) : u);
            }
        if (p.b) {
            w.load(p.b, p.w_type, t, T, p.cols);
            w.widen(p.w_type);
#pragma unroll
            for (int e = 0; e < E; ++e)
#pragma unroll
                for (int i = 0; i < V; ++i) h.set(e, i, h.get(e, i) + w.get(e, i));
        }
        h.store(row_of(p.y, p.y_type, row, p.cols), p.y_type, t, T, p.cols);
    }
}

// kSum: the sum's own gradient dh is added to dx.  p.part: the CTA's column sums
// [gridDim][2][cols] (dw, db), or null when no weight gradient is wanted.
template <int V, int E, int W, bool kSum>
__global__ void __launch_bounds__(cta_threads(W)) norm_bwd_kernel(NormParams p) {
    constexpr int T = W * 32;
    __shared__ float red[2][W][2];
    int slot = 0;
    const int t = W == 1 ? (threadIdx.x & 31) : threadIdx.x;
    const long long first = W == 1 ? (long long)blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x;
    float dw[E][V] = {}, db[E][V] = {};
    for (long long row = first; row < p.rows; row += (long long)gridDim.x * cta_rows(W)) {
        Row<V, E> u, g, a;
        u.load(row_of(p.x, p.x_type, row, p.x_stride), p.x_type, t, T, p.cols);
        g.load(row_of(p.dy, p.y_type, row, p.dy_stride), p.y_type, t, T, p.cols);
        if constexpr (kSum) a.load(row_of(p.dh, p.x_type, row, p.dh_stride), p.x_type, t, T, p.cols);
        const float mean = __ldg(p.mean + row), rstd = __ldg(p.rstd + row);
        u.widen(p.x_type);
        g.widen(p.y_type);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const bool in = (e * T + t) * V < p.cols;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float v = in ? (u.get(e, i) - mean) * rstd : 0.0f;
                u.set(e, i, v);
                dw[e][i] = fmaf(g.get(e, i), v, dw[e][i]);
                db[e][i] += g.get(e, i);
            }
        }
        if (p.w) {
            Row<V, E> w;
            w.load(p.w, p.w_type, t, T, p.cols);
            w.widen(p.w_type);
#pragma unroll
            for (int e = 0; e < E; ++e)
#pragma unroll
                for (int i = 0; i < V; ++i) g.set(e, i, g.get(e, i) * w.get(e, i));
        }
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                s[0] += g.get(e, i);
                s[1] = fmaf(g.get(e, i), u.get(e, i), s[1]);
            }
        row_sum<W, 2>(s, red, slot);
        const float c1 = s[0] / (float)p.cols, c2 = s[1] / (float)p.cols;
        if constexpr (kSum) a.widen(p.x_type);
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float v = rstd * (g.get(e, i) - c1 - u.get(e, i) * c2);
                g.set(e, i, kSum ? v + a.get(e, i) : v);
            }
        if (p.dx) g.store(row_of(p.dx, p.x_type, row, p.cols), p.x_type, t, T, p.cols);
        if (p.dd) g.store(row_of(p.dd, p.d_type, row, p.cols), p.d_type, t, T, p.cols);
    }
    if (!p.part) return;
    float* out = p.part + (long long)blockIdx.x * 2 * p.cols;
    if constexpr (W == 1) {
        // join the eight warps' sums, one array after the other
        __shared__ float join[8][T * V * E];
        for (int k = 0; k < 2; ++k) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < E; ++e)
#pragma unroll
                for (int i = 0; i < V; ++i) join[threadIdx.x >> 5][(e * T + t) * V + i] = k ? db[e][i] : dw[e][i];
            __syncthreads();
            for (int c = threadIdx.x; c < p.cols; c += 256) {
                float s = 0.0f;
#pragma unroll
                for (int w = 0; w < 8; ++w) s += join[w][c];
                out[k * p.cols + c] = s;
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int col = (e * T + t) * V;
            if (col < p.cols) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    out[col + i] = dw[e][i];
                    out[p.cols + col + i] = db[e][i];
                }
            }
        }
    }
}

// dw / db (blockIdx.y) of 32 columns: kReduceLanes partial rows side by side,
// then a fixed tree over them.
__global__ void __launch_bounds__(32 * kReduceLanes) norm_cols_kernel(const float* part, int nparts, int cols, void* dw,
                                                                       void* db, int type) {
    __shared__ float s[kReduceLanes][33];
    void* out = blockIdx.y ? db : dw;
    if (!out) return;
    const int c = blockIdx.x * 32 + threadIdx.x;
    float v = 0.0f;
    if (c < cols) {
        const float* src = part + (long long)blockIdx.y * cols + c;
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
};

// Row layout by width: the smallest of these that holds the row.  Vectors of
// four need widths, strides and addresses that are multiples of four elements.
constexpr Shape kShapes[] = {{4, 1, 1}, {4, 2, 1}, {4, 3, 1}, {4, 4, 1},  {4, 6, 1},  {4, 8, 1},  {4, 4, 4},
                             {4, 4, 8}, {4, 8, 8}, {4, 8, 16}, {1, 8, 1}, {1, 32, 1}, {1, 16, 8}, {1, 32, 16}};
constexpr int kNumShapes = sizeof(kShapes) / sizeof(kShapes[0]);

int pick_shape(int cols, bool vec) {
    for (int i = 0; i < kNumShapes; ++i) {
        const Shape s = kShapes[i];
        if ((s.v == 4) == vec && s.v * s.e * s.w * 32 >= cols) return i;
    }
    return kNumShapes - 1;
}

using Kernel = void (*)(NormParams);

template <int I>
constexpr Kernel fwd_of(bool delta) {
    constexpr Shape s = kShapes[I];
    return delta ? (Kernel)norm_fwd_kernel<s.v, s.e, s.w, true> : (Kernel)norm_fwd_kernel<s.v, s.e, s.w, false>;
}
template <int I>
constexpr Kernel bwd_of(bool sum) {
    constexpr Shape s = kShapes[I];
    return sum ? (Kernel)norm_bwd_kernel<s.v, s.e, s.w, true> : (Kernel)norm_bwd_kernel<s.v, s.e, s.w, false>;
}

#define CIMEKV_NORM_TABLE(F, flag) \
    {F<0>(flag), F<1>(flag), F<2>(flag), F<3>(flag), F<4>(flag), F<5>(flag), F<6>(flag), \
     F<7>(flag), F<8>(flag), F<9>(flag), F<10>(flag), F<11>(flag), F<12>(flag), F<13>(flag)}
const Kernel kFwd[2][kNumShapes] = {CIMEKV_NORM_TABLE(fwd_of, false), CIMEKV_NORM_TABLE(fwd_of, true)};
const Kernel kBwd[2][kNumShapes] = {CIMEKV_NORM_TABLE(bwd_of, false), CIMEKV_NORM_TABLE(bwd_of, true)};

int sm_count(int* sms) {
    int dev;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        return fail(CIMEKV_ECUDA, "cannot read the device's SM count");
    return CIMEKV_OK;
}

// CTAs per SM that the row loops are spread over (both directions keep at least
// this many resident).
int ctas_per_sm(const Shape& s) { return s.w == 1 ? 4 : s.w == 4 ? 8 : s.w == 8 ? 4 : 2; }

long long grid_size(long long rows, const Shape& s, int sms) {
    const long long need = (rows + cta_rows(s.w) - 1) / cta_rows(s.w);
    const long long most = (long long)sms * ctas_per_sm(s);
    return need < most ? need : most;
}

bool valid_type(int t) { return t == CIMEKV_F32 || t == CIMEKV_BF16 || t == CIMEKV_F16; }

// Whether rows of `p` can be moved in vectors of four elements.
bool vec_ok(const void* p, int type, long long stride) {
    return !p || (((uintptr_t)p % (4 * (size_t)type_bytes(type))) == 0 && stride % 4 == 0);
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
    const bool vec = cols % 4 == 0 && vec_ok(x, x_type, x_stride) && vec_ok(delta, delta_type, delta_stride) &&
                     vec_ok(h, x_type, cols) && vec_ok(y, y_type, cols) && vec_ok(weight, w_type, 0) &&
                     vec_ok(bias, w_type, 0);
    const int i = pick_shape(cols, vec);
    int sms;
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
    p.eps = eps;
    if ((rc = cimekv_internal_no_pending_error())) return rc;
    kFwd[delta != nullptr][i]<<<(unsigned)grid_size(rows, kShapes[i], sms), cta_threads(kShapes[i].w), 0,
                                (cudaStream_t)stream>>>(p);
    return launched("norm_fwd_kernel");
}

// The widest grid any layout takes, so that the size does not depend on
// addresses (which decide between the vector and the scalar layout).
extern "C" size_t cimekv_layer_norm_workspace_bytes(long long rows, int cols) {
    if (rows <= 0 || cols < 1 || cols > kMaxCols) return 0;
    int sms;
    if (sm_count(&sms)) return 0;
    long long most = 0;
    for (const bool vec : {false, true}) {
        const long long g = grid_size(rows, kShapes[pick_shape(cols, vec)], sms);
        if (g > most) most = g;
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
        const bool vec = cols % 4 == 0 && vec_ok(h, x_type, h_stride) && vec_ok(dy, y_type, dy_stride) &&
                         vec_ok(dh, x_type, dh_stride) && vec_ok(dx, x_type, cols) &&
                         vec_ok(ddelta, delta_type, cols) && vec_ok(weight, w_type, 0);
        const int i = pick_shape(cols, vec);
        int sms;
        if ((rc = sm_count(&sms))) return rc;
        const long long grid = grid_size(rows, kShapes[i], sms);
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
        if ((rc = cimekv_internal_no_pending_error())) return rc;
        kBwd[dh != nullptr][i]<<<(unsigned)grid, cta_threads(kShapes[i].w), 0, s>>>(p);
        if ((rc = launched("norm_bwd_kernel"))) return rc;
        nparts = (int)grid;
    } else if ((rc = cimekv_internal_no_pending_error())) {
        return rc;
    }
    if (!want_w) return CIMEKV_OK;
    // no rows: the sums over none of them are zero
    norm_cols_kernel<<<dim3((unsigned)(cols + 31) / 32, 2), dim3(32, kReduceLanes), 0, s>>>(
        static_cast<const float*>(workspace), nparts, cols, dw, db, w_type);
    return launched("norm_cols_kernel");
}
