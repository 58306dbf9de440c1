// newton_schulz.cu — orthogonalisation of update matrices by Newton-Schulz
// products on the tensor cores, and the Muon optimiser step around it.
//
// With X0 = G / max(|G|_F, eps), m rows and n >= m columns (a tall G is worked on
// transposed), each step is
//
//   A = X X^T,   P = a I + b A + c A A,   X <- P X
//
// so the singular values s of X go through s (a + b s^2 + c s^4) and close in on
// one band around 1, while the singular vectors stay.  All three are products of
// matrices; everything elementwise sits in their epilogues.
//
// Precision.  A singular value far below the largest grows by up to a per step
// (x 485 in five steps), and so does any rounding noise in its direction: with
// operands rounded to 11 bits the result of a low-rank update is off by 1e-2, more
// than the half step of a bf16 result.  X, A and P are therefore held as pairs of
// fp16 planes, value * 2^12 = hi + lo (22 bits; the iteration keeps singular
// values of X and A below 2 and of P below 15, checked on the host from the
// coefficients, so the fixed scale neither overflows nor loses small elements), and a
// product is hi hi + hi lo + lo hi, accumulated in fp32 in tensor memory: three
// tensor core products, closer to the exact result than fp32 FMAs.
//
// A and P are symmetric: only tiles on and below the diagonal are computed, the
// epilogue stores each tile and its mirror image.

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <mutex>
#include <utility>

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

int launched(const char* what) {
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) return CIMEKV_OK;
    char msg[256];
    snprintf(msg, sizeof(msg), "%s: %s", what, cudaGetErrorString(e));
    return fail(CIMEKV_ECUDA, msg);
}

constexpr float kScale = 4096.0f;  // fp16 planes hold value * 2^12
constexpr int kTile = 128;         // rows (and right-hand rows) that one CTA stages
constexpr int kK = 64;             // depth of one stage: 64 halves = one 128-byte swizzle row
constexpr int kStages = 3;
constexpr int kChunk = 2;                   // stages summed in tensor memory before fp32 registers take over
constexpr int kOperand = kTile * kK * 2;    // bytes of one operand plane in a stage
constexpr int kStageBytes = 4 * kOperand;   // left hi, left lo, right hi, right lo
constexpr int kEpilogueWarps = 8;
constexpr int kGemmThreads = (kEpilogueWarps + 2) * 32;  // and a copy warp, a product warp
constexpr int kSmemBytes = kStages * kStageBytes + 1024;
constexpr int kMaxTable = CIMEKV_MUON_MAX_MATRICES;
constexpr int kChunks = 64;                 // partial norms per matrix

// ------------------------------------------------------------- PTX pieces --

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

// Waits for the phase of `parity` to end, for about a second at most: a wait
// that runs out means a lost copy, and its tile is poisoned instead of hanging.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity) {
    for (int i = 0; i < (1 << 20); ++i) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 1000;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
        if (done) return true;
    }
    return false;
}

// Address of the same shared variable in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

// One box of a plane (rows of 64 halves, 16-byte units swizzled) into this CTA;
// the bytes are counted on `bar`, which is the first CTA's in a pair.
template <bool kPair>
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    if constexpr (kPair)
        asm volatile(
            "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
            "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
            "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
            : "memory");
}

// Shared-memory operand descriptors, 128-byte swizzle.  Rows along K (a plane's
// row is an operand row): groups of 8 rows are 1024 bytes apart.  Rows along the
// other axis (a plane's row is a K index): 8 K indexes are 1024 bytes, the next 64
// elements of a row lie one box (8192 bytes) further.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, uint32_t leading, uint32_t stride) {
    return (uint64_t)((addr & 0x3ffff) >> 4) | (uint64_t)(leading >> 4) << 16 | (uint64_t)(stride >> 4) << 32 |
           (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

template <bool kPair>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (kPair)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
}
// Arrives on `bar` (in both CTAs of a pair) when the products issued so far are done.
template <bool kPair>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    if constexpr (kPair)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
            "h"((uint16_t)3)
            : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
template <bool kPair>
__device__ __forceinline__ void tmem_alloc(uint32_t slot, uint32_t columns) {
    if constexpr (kPair) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
}
template <bool kPair>
__device__ __forceinline__ void tmem_free(uint32_t tmem, uint32_t columns) {
    if constexpr (kPair)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
    else
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
}

__device__ __forceinline__ void tmem_load32(uint32_t addr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// ------------------------------------------------------------------ types ---

__device__ __forceinline__ float load_as_float(const void* p, int type, long long i) {
    if (type == CIMEKV_F32) return static_cast<const float*>(p)[i];
    if (type == CIMEKV_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_float(void* p, int type, long long i, float v) {
    if (type == CIMEKV_F32) static_cast<float*>(p)[i] = v;
    else if (type == CIMEKV_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
    else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// The matrices of one call: either `table` pointers or one base and a stride.
struct Matrices {
    const void* base;
    long long batch_stride, row_stride;  // elements
    int type;
    int tabled;
    void* table[kMaxTable];

    __device__ __forceinline__ const void* at(int b) const {
        if (tabled) return table[b];
        return static_cast<const char*>(base) + b * batch_stride * (type == CIMEKV_F32 ? 4 : 2);
    }
};

struct PrepParams {
    Matrices g;
    Matrices mom;       // momenta (fp32, contiguous), table only; tabled = 0: none
    float beta;
    int nesterov;
    int rows, cols;     // of G
    int transposed;     // rows > cols
    int pitch;          // of the planes, elements
    long long plane;    // elements from the hi to the lo plane
    float eps;
    double* part;       // [batch][kChunks]
    __half* x;
};

// The update before orthogonalisation: G itself, or the (Nesterov) momentum after
// its own update m <- beta m + (1 - beta) g.
__device__ __forceinline__ float update_of(const PrepParams& p, float g, float m) {
    return p.nesterov ? fmaf(p.beta, m, (1.0f - p.beta) * g) : m;
}

// Momentum update and the partial sums of squares of one matrix: kChunks CTAs
// per matrix, in doubles (squares of fp32 values neither overflow nor vanish),
// added in a fixed order.
__global__ void __launch_bounds__(256) ns_norm_kernel(const __grid_constant__ PrepParams p) {
    const int b = blockIdx.y;
    const void* g = p.g.at(b);
    float* mom = p.mom.tabled ? static_cast<float*>(p.mom.table[b]) : nullptr;
    const long long total = (long long)p.rows * p.cols;
    double s = 0.0;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += kChunks * 256) {
        const long long r = i / p.cols, c = i - r * p.cols;
        float v = load_as_float(g, p.g.type, r * p.g.row_stride + c);
        if (mom) {
            const float m = fmaf(p.beta, mom[i], (1.0f - p.beta) * v);
            mom[i] = m;
            v = update_of(p, v, m);
        }
        s += (double)v * (double)v;
    }
    __shared__ double red[8];
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; ++w) s += red[w];
        p.part[(long long)b * kChunks + blockIdx.x] = s;
    }
}

__device__ __forceinline__ void split(float scaled, __half& hi, __half& lo) {
    hi = __float2half_rn(scaled);
    lo = __float2half_rn(scaled - __half2float(hi));
}

// X0 as pairs of planes, transposed where G is tall: 32 x 32 tiles through
// shared memory, so that reads and writes are both along rows.
__global__ void __launch_bounds__(256) ns_prepare_kernel(const __grid_constant__ PrepParams p) {
    __shared__ float tile[32][33];
    __shared__ float factor;
    const int b = blockIdx.z;
    if (threadIdx.x == 0) {
        double s = 0.0;
        for (int i = 0; i < kChunks; ++i) s += p.part[(long long)b * kChunks + i];
        const double norm = sqrt(s);
        factor = (float)((double)kScale / (norm > (double)p.eps || norm != norm ? norm : (double)p.eps));
    }
    const void* g = p.g.at(b);
    const float* mom = p.mom.tabled ? static_cast<const float*>(p.mom.table[b]) : nullptr;
    const int r0 = blockIdx.y * 32, c0 = blockIdx.x * 32;
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    for (int k = ty; k < 32; k += 8) {
        const int r = r0 + k, c = c0 + tx;
        if (r < p.rows && c < p.cols) {
            float v = load_as_float(g, p.g.type, r * p.g.row_stride + c);
            if (mom) v = update_of(p, v, mom[(long long)r * p.cols + c]);
            tile[k][tx] = v;
        }
    }
    __syncthreads();
    const int m = p.transposed ? p.cols : p.rows, n = p.transposed ? p.rows : p.cols;
    __half* x = p.x + (long long)b * m * p.pitch;
    for (int k = ty; k < 32; k += 8) {
        const int r = (p.transposed ? c0 : r0) + k, c = (p.transposed ? r0 : c0) + tx;
        if (r < m && c < n) {
            __half hi, lo;
            split((p.transposed ? tile[tx][k] : tile[k][tx]) * factor, hi, lo);
            x[(long long)r * p.pitch + c] = hi;
            x[p.plane + (long long)r * p.pitch + c] = lo;
        }
    }
}

// ---------------------------------------------------------------- products --

enum Mode { kGram = 0, kPoly = 1, kApply = 2, kResult = 3 };

struct GemmParams {
    int rows, cols, depth;  // of the product
    int batch;
    __half* out;            // planes of the result (kGram, kPoly, kApply)
    long long out_plane;    // elements from hi to lo
    int out_pitch;
    const __half* a;        // planes of A (kPoly)
    float ca, cb, cc;
    // kResult: where X goes
    int transposed;
    Matrices dst;           // results, or parameters to update in place
    int update;             // parameters: p <- p (1 - lr decay) - lr scale X
    float lr, decay, scale;
    const float* lr_dev;
};

// Tile (i, j) of the lower triangle, row by row.
__device__ __forceinline__ void triangle(int t, int& i, int& j) {
    i = (int)((sqrtf(8.0f * (float)t + 1.0f) - 1.0f) * 0.5f);
    while ((i + 1) * (i + 2) / 2 <= t) ++i;
    while (i * (i + 1) / 2 > t) --i;
    j = t - i * (i + 1) / 2;
}

// 32 columns of one row of a finished tile: `v` are sums of scaled products.
template <int M>
__device__ __forceinline__ void finish(const GemmParams& p, float (&v)[32], int b, int r, int cb, bool mirrored, float lr) {
    if constexpr (M == kResult) {
        void* dst = const_cast<void*>(p.dst.at(b));
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            if (cb + i >= p.cols) break;
            const long long at = p.transposed ? (long long)(cb + i) * p.rows + r : (long long)r * p.cols + cb + i;
            float o = v[i] * (1.0f / (kScale * kScale));
            if (p.update) {
                const float w = load_as_float(dst, p.dst.type, at);
                o = fmaf(-lr * p.scale, o, fmaf(-lr * p.decay, w, w));
            }
            store_float(dst, p.dst.type, at, o);
        }
    } else {
        const long long mat = (long long)b * p.rows * p.out_pitch;
        uint32_t hi[16], lo[16];
        const __half* ah = p.a + mat + (long long)r * p.out_pitch + cb;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            float o = v[i] * (1.0f / kScale);
            if (M == kPoly) {
                const bool in = cb + i < p.cols;
                const float a = in ? __half2float(ah[i]) + __half2float(ah[p.out_plane + i]) : 0.0f;
                o = fmaf(p.cc, o, p.cb * a) + (r == cb + i ? p.ca * kScale : 0.0f);
            }
            v[i] = o;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            __half h0, l0, h1, l1;
            split(v[2 * i], h0, l0);
            split(v[2 * i + 1], h1, l1);
            hi[i] = (uint32_t)__half_as_ushort(h0) | (uint32_t)__half_as_ushort(h1) << 16;
            lo[i] = (uint32_t)__half_as_ushort(l0) | (uint32_t)__half_as_ushort(l1) << 16;
        }
        __half* oh = p.out + mat + (long long)r * p.out_pitch + cb;
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // the pitch is a multiple of 8: a group that begins inside ends inside
            if (cb + 8 * i < p.cols) {
                *reinterpret_cast<uint4*>(oh + 8 * i) = make_uint4(hi[4 * i], hi[4 * i + 1], hi[4 * i + 2], hi[4 * i + 3]);
                *reinterpret_cast<uint4*>(oh + p.out_plane + 8 * i) =
                    make_uint4(lo[4 * i], lo[4 * i + 1], lo[4 * i + 2], lo[4 * i + 3]);
            }
        }
        if (M <= kPoly && mirrored) {
            __half* mirror = p.out + mat + (long long)cb * p.out_pitch + r;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                if (cb + i < p.cols) {
                    const uint32_t h = hi[i / 2] >> (16 * (i & 1)), l = lo[i / 2] >> (16 * (i & 1));
                    mirror[(long long)i * p.out_pitch] = __ushort_as_half((unsigned short)h);
                    mirror[p.out_plane + (long long)i * p.out_pitch] = __ushort_as_half((unsigned short)l);
                }
            }
        }
    }
}

// A persistent loop over output tiles: 128 x 128 by one CTA, or 256 x 256 by a
// pair of CTAs whose tensor cores work as one (each stages 128 rows of either
// operand, holds its 128 rows of the result, and the first CTA issues).  One warp
// copies stages ahead, one issues products, eight collect.
//
// The tensor core adds into fp32 accumulators by cutting off, not by rounding:
// over a long depth that is a drift of half a step per addition.  So a tile's
// depth is summed in chunks of kChunk stages that alternate between two
// accumulators, the small cross products of a stage first, and the collecting
// warps add the chunks in registers with round-to-nearest while the next chunk
// runs.  The same two accumulators let the next tile start while the last one is
// stored.
template <int M, bool kPair>
__global__ void __launch_bounds__(kGemmThreads, 1) ns_gemm_kernel(const __grid_constant__ CUtensorMap left,
                                                                  const __grid_constant__ CUtensorMap right,
                                                                  const __grid_constant__ GemmParams p) {
    constexpr int kRanks = kPair ? 2 : 1;
    constexpr int kSide = kTile * kRanks;          // output tile side, and columns of an accumulator
    constexpr int kWarpCols = kSide / 2;           // columns a collecting warp holds
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[2 * kStages + 5];
    __shared__ uint32_t tmem_slot;
    const uint32_t stages = (smem_addr(smem_raw) + 1023) & ~1023u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = kPair ? cluster_rank() : 0;
    const uint32_t full = smem_addr(bars), empty = full + 8 * kStages, acc_full = full + 16 * kStages,
                   acc_empty = acc_full + 16, drained = acc_full + 32;
    const int ni = (p.rows + kSide - 1) / kSide, nj = (p.cols + kSide - 1) / kSide;
    const int per_matrix = M <= kPoly ? ni * (ni + 1) / 2 : ni * nj;
    const long long tiles = (long long)per_matrix * p.batch;
    const int ksteps = (p.depth + kK - 1) / kK;
    const int step = gridDim.x / kRanks, first = blockIdx.x / kRanks;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full + 8 * s, 1);
            mbar_init(empty + 8 * s, 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(acc_full + 8 * s, 1);
            mbar_init(acc_empty + 8 * s, kEpilogueWarps * kRanks);
        }
        mbar_init(drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kEpilogueWarps + 1) tmem_alloc<kPair>(smem_addr(&tmem_slot), 2 * kSide);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if constexpr (kPair) cluster_sync();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_slot;

    const auto place = [&](long long t, int& b, int& row0, int& col0) {
        b = (int)(t / per_matrix);
        const int at = (int)(t - (long long)b * per_matrix);
        int i, j;
        if (M <= kPoly) {
            triangle(at, i, j);
        } else {
            i = at / nj;
            j = at - i * nj;
        }
        row0 = i * kSide;
        col0 = j * kSide;
    };

    if (warp == kEpilogueWarps) {
        if (lane == 0) {
            const uint32_t count_at = kPair ? cluster_addr(full, 0) : full;
            bool ok = true;
            int fill = 0;
            for (long long t = first; t < tiles && ok; t += step) {
                int b, row0, col0;
                place(t, b, row0, col0);
                row0 += (int)rank * kTile;
                col0 += (int)rank * kTile;
                for (int k = 0; k < ksteps; ++k, ++fill) {
                    const int s = fill % kStages;
                    if (fill >= kStages && !(ok = mbar_wait(empty + 8 * s, (fill / kStages - 1) & 1))) break;
                    const uint32_t base = stages + s * kStageBytes, bar = count_at + 8 * s;
                    if (rank == 0) mbar_expect(full + 8 * s, kRanks * kStageBytes);
#pragma unroll
                    for (int plane = 0; plane < 2; ++plane) {
                        const int z = plane * p.batch + b;
                        const uint32_t l = base + plane * kOperand, r = base + (2 + plane) * kOperand;
                        tma_box<kPair>(l, &left, k * kK, row0, z, bar);
                        if (M <= kPoly) {
                            tma_box<kPair>(r, &right, k * kK, col0, z, bar);
                        } else {
                            tma_box<kPair>(r, &right, col0, k * kK, z, bar);
                            tma_box<kPair>(r + kOperand / 2, &right, col0 + 64, k * kK, z, bar);
                        }
                    }
                }
            }
            // no copy may still be in flight when the CTA leaves (a pair's are all counted in the first)
            if (rank == 0)
                for (int s = 0; s < kStages; ++s) {
                    const int fills = (fill - s + kStages - 1) / kStages;
                    if (fills > 0) mbar_wait(full + 8 * s, (fills - 1) & 1);
                }
        }
    } else if (warp == kEpilogueWarps + 1) {
        if (lane == 0 && rank == 0) {
            // D fp32, A and B fp16; right operand along K (0) or along its own axis (1)
            const uint32_t idesc = 1u << 4 | (M <= kPoly ? 0u : 1u << 16) | (uint32_t)(kSide / 8) << 17 |
                                   (uint32_t)(kSide / 16) << 24;
            bool ok = true;
            int fill = 0, chunk = 0;
            for (long long t = first; t < tiles && ok; t += step) {
                for (int k = 0; k < ksteps && ok; ++chunk) {
                    const int buf = chunk & 1;
                    if (chunk >= 2 && !(ok = mbar_wait(acc_empty + 8 * buf, (chunk / 2 - 1) & 1))) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t d = tmem + buf * kSide;
                    const int end = min(k + kChunk, ksteps);
                    for (bool fresh = true; k < end; ++k, ++fill, fresh = false) {
                        const int s = fill % kStages;
                        if (!(ok = mbar_wait(full + 8 * s, (fill / kStages) & 1))) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const uint32_t base = stages + s * kStageBytes;
                        const auto desc_l = [&](int plane, int q) {
                            return operand_desc(base + plane * kOperand + q * 32, 16, 1024);
                        };
                        const auto desc_r = [&](int plane, int q) {
                            return M <= kPoly ? operand_desc(base + (2 + plane) * kOperand + q * 32, 16, 1024)
                                              : operand_desc(base + (2 + plane) * kOperand + q * 2048, 8192, 1024);
                        };
#pragma unroll
                        for (int q = 0; q < kK / 16; ++q) {
                            mma_f16<kPair>(d, desc_l(0, q), desc_r(1, q), idesc, !(fresh && q == 0));
                            mma_f16<kPair>(d, desc_l(1, q), desc_r(0, q), idesc, 1);
                        }
#pragma unroll
                        for (int q = 0; q < kK / 16; ++q) mma_f16<kPair>(d, desc_l(0, q), desc_r(0, q), idesc, 1);
                        mma_commit<kPair>(empty + 8 * s);
                    }
                    if (ok) mma_commit<kPair>(acc_full + 8 * buf);
                }
            }
            mma_commit<kPair>(drained);  // no product may still read shared memory when the CTAs leave
            mbar_wait(drained, 0);
        }
    } else {
        const int quarter = warp & 3, half = warp >> 2;
        const uint32_t empty_at = kPair ? cluster_addr(acc_empty, 0) : acc_empty;
        const float lr = M == kResult && p.update ? (p.lr_dev ? *p.lr_dev : p.lr) : 0.0f;
        bool ok = true;
        int chunk = 0;
        for (long long t = first; t < tiles; t += step) {
            int b, row0, col0;
            place(t, b, row0, col0);
            const int r = row0 + (int)rank * kTile + quarter * 32 + lane;
            const bool mirrored = row0 != col0;
            col0 += half * kWarpCols;
            float acc[kWarpCols / 32][32];
#pragma unroll
            for (int g = 0; g < kWarpCols / 32; ++g)
#pragma unroll
                for (int i = 0; i < 32; ++i) acc[g][i] = 0.0f;
            for (int k = 0; k < ksteps; k += kChunk, ++chunk) {
                const int buf = chunk & 1;
                ok = ok && mbar_wait(acc_full + 8 * buf, (chunk / 2) & 1);
                __syncwarp();
                if (!__all_sync(0xffffffffu, ok)) {
                    ok = false;
                    continue;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t src = tmem + ((uint32_t)(quarter * 32) << 16) + buf * kSide + half * kWarpCols;
#pragma unroll
                for (int g = 0; g < kWarpCols / 32; ++g) {
                    float v[32];
                    tmem_load32(src + g * 32, v);
#pragma unroll
                    for (int i = 0; i < 32; ++i) acc[g][i] += v[i];
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(empty_at + 8 * buf);
            }
            if (!ok) {  // a lost copy or product shows as NaN, it never passes for a result
#pragma unroll
                for (int g = 0; g < kWarpCols / 32; ++g)
#pragma unroll
                    for (int i = 0; i < 32; ++i) acc[g][i] = __int_as_float(0x7fffffff);
            }
            if (r < p.rows) {
#pragma unroll
                for (int g = 0; g < kWarpCols / 32; ++g)
                    if (col0 + g * 32 < p.cols) finish<M>(p, acc[g], b, r, col0 + g * 32, mirrored, lr);
            }
            __syncwarp();
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if constexpr (kPair) cluster_sync();  // the other CTA may still signal or read here
    if (warp == kEpilogueWarps + 1) {
        __syncwarp();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        tmem_free<kPair>(tmem, 2 * kSide);
    }
}

// ------------------------------------------------------------------ host ----

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int encoder(EncodeFn* out) {
    static std::mutex mutex;
    static EncodeFn fn = nullptr;
    std::lock_guard<std::mutex> lock(mutex);
    if (!fn) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess || !p)
            return fail(CIMEKV_ECUDA, "the driver has no cuTensorMapEncodeTiled");
        fn = reinterpret_cast<EncodeFn>(p);
    }
    *out = fn;
    return CIMEKV_OK;
}

// Planes [2 * batch][rows][cols] of a given pitch, boxes of 64 columns, zeros outside.
int plane_map(EncodeFn encode, CUtensorMap* map, __half* base, int batch, int rows, int cols, int pitch, int box_rows) {
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)2 * batch};
    const cuuint64_t strides[2] = {(cuuint64_t)pitch * 2, (cuuint64_t)pitch * 2 * rows};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1}, step[3] = {1, 1, 1};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, base, dims, strides, box, step,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? CIMEKV_OK : fail(CIMEKV_ECUDA, "cuTensorMapEncodeTiled refused a plane");
}

// Workspace: partial norms, X twice, A, P (pairs of planes each).
struct Layout {
    int m, n, xp, ap;               // sides (m <= n) and pitches
    size_t part, x0, x1, a, p, bytes;
    long long x_plane, a_plane;     // elements

    Layout(int batch, int rows, int cols) {
        m = rows < cols ? rows : cols;
        n = rows < cols ? cols : rows;
        xp = (n + 7) / 8 * 8;
        ap = (m + 7) / 8 * 8;
        x_plane = (long long)batch * m * xp;
        a_plane = (long long)batch * m * ap;
        size_t at = 0;
        const auto take = [&at](size_t b) {
            const size_t here = at;
            at += (b + 255) / 256 * 256;
            return here;
        };
        part = take((size_t)batch * kChunks * sizeof(double));
        x0 = take((size_t)x_plane * 4);
        x1 = take((size_t)x_plane * 4);
        a = take((size_t)a_plane * 4);
        p = take((size_t)a_plane * 4);
        bytes = at;
    }
};

constexpr int kMaxSide = CIMEKV_ORTHOGONALIZE_MAX_SIDE;

int check_iteration(int batch, int rows, int cols, int steps, float a, float b, float c, float eps) {
    if (batch < 0 || rows < 0 || cols < 0) return fail(CIMEKV_EINVAL_SHAPE, "negative size");
    if (rows > kMaxSide || cols > kMaxSide || batch > 65535)
        return fail(CIMEKV_EINVAL_SHAPE, "orthogonalize: sides of at most 32768, at most 65535 matrices");
    if (steps < 1 || steps > 64) return fail(CIMEKV_EINVAL_SHAPE, "orthogonalize: 1 to 64 steps");
    if (!(eps > 0.0f)) return fail(CIMEKV_EINVAL_SHAPE, "eps must be > 0");
    if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c))
        return fail(CIMEKV_EINVAL_SHAPE, "orthogonalize: coefficients must be finite");
    // Largest singular value over the steps, and largest |a + b l + c l^2| on its
    // range: both must fit the planes' fixed scale (16 / 2^12-scaled fp16).
    double s = 1.001;
    for (int k = 0; k < steps; ++k) {
        double next = 0.0, poly = 0.0;
        for (int i = 0; i <= 1024; ++i) {
            const double t = s * i / 1024.0, q = a + (b + c * t * t) * t * t;
            next = std::fmax(next, std::fabs(t * q));
            poly = std::fmax(poly, std::fabs(q));
        }
        s = next * 1.001;
        if (!(s <= 3.9 && poly <= 15.0))
            return fail(CIMEKV_EINVAL_SHAPE,
                        "orthogonalize: these coefficients let singular values grow beyond 3.9 (or their factor beyond 15)");
    }
    return CIMEKV_OK;
}

int sm_count(int* sms) {
    int dev;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        return fail(CIMEKV_ECUDA, "cannot read the device's SM count");
    return CIMEKV_OK;
}

long long tile_count(int mode, int side, const GemmParams& p) {
    const long long ni = (p.rows + side - 1) / side, nj = (p.cols + side - 1) / side;
    return (mode <= kPoly ? ni * (ni + 1) / 2 : ni * nj) * p.batch;
}

template <int M, bool kPair>
int launch_as(const CUtensorMap& l, const CUtensorMap& r, const GemmParams& p, int sms, cudaStream_t s) {
    cudaError_t e = cudaFuncSetAttribute(ns_gemm_kernel<M, kPair>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
    if (e != cudaSuccess) return fail(CIMEKV_ECUDA, cudaGetErrorString(e));
    constexpr int ranks = kPair ? 2 : 1;
    const long long tiles = tile_count(M, kTile * ranks, p), most = sms / ranks;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles < most ? tiles : most) * ranks);
    cfg.blockDim = dim3(kGemmThreads);
    cfg.dynamicSmemBytes = kSmemBytes;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = kPair ? 1 : 0;
    e = cudaLaunchKernelEx(&cfg, ns_gemm_kernel<M, kPair>, l, r, p);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return fail(CIMEKV_ECUDA, cudaGetErrorString(e));
    }
    return CIMEKV_OK;
}

// Pairs once single tiles would fill every SM anyway: the larger tile halves
// the operand traffic; below that the smaller one spreads over more SMs.
template <int M>
int launch_gemm(const CUtensorMap& l, const CUtensorMap& r, const GemmParams& p, int sms, cudaStream_t s) {
    return tile_count(M, kTile, p) > sms ? launch_as<M, true>(l, r, p, sms, s) : launch_as<M, false>(l, r, p, sms, s);
}

// Everything after the arguments are checked: norms, X0, the steps, the result.
int run(PrepParams& prep, GemmParams& out, int batch, int rows, int cols, int steps, float a, float b, float c,
        uint8_t* ws, cudaStream_t s) {
    const Layout lay(batch, rows, cols);
    EncodeFn encode;
    int rc;
    int sms;
    if ((rc = encoder(&encode)) || (rc = sm_count(&sms))) return rc;
    __half* x[2] = {reinterpret_cast<__half*>(ws + lay.x0), reinterpret_cast<__half*>(ws + lay.x1)};
    __half* am = reinterpret_cast<__half*>(ws + lay.a);
    __half* pm = reinterpret_cast<__half*>(ws + lay.p);
    // X as rows along K (Gram) and as the right operand whose rows are K (apply)
    CUtensorMap xmap[2], xright[2], amap, pmap;
    for (int i = 0; i < 2; ++i) {
        if ((rc = plane_map(encode, &xmap[i], x[i], batch, lay.m, lay.n, lay.xp, kTile))) return rc;
        if ((rc = plane_map(encode, &xright[i], x[i], batch, lay.m, lay.n, lay.xp, kK))) return rc;
    }
    if ((rc = plane_map(encode, &amap, am, batch, lay.m, lay.m, lay.ap, kTile))) return rc;
    if ((rc = plane_map(encode, &pmap, pm, batch, lay.m, lay.m, lay.ap, kTile))) return rc;

    prep.rows = rows;
    prep.cols = cols;
    prep.transposed = rows > cols;
    prep.pitch = lay.xp;
    prep.plane = lay.x_plane;
    prep.part = reinterpret_cast<double*>(ws + lay.part);
    prep.x = x[0];
    if ((rc = cimekv_internal_no_pending_error())) return rc;
    ns_norm_kernel<<<dim3(kChunks, batch), 256, 0, s>>>(prep);
    if ((rc = launched("ns_norm_kernel"))) return rc;
    ns_prepare_kernel<<<dim3((cols + 31) / 32, (rows + 31) / 32, batch), 256, 0, s>>>(prep);
    if ((rc = launched("ns_prepare_kernel"))) return rc;

    GemmParams g = {};
    g.batch = batch;
    g.ca = a;
    g.cb = b;
    g.cc = c;
    for (int k = 0; k < steps; ++k) {
        g.rows = g.cols = lay.m;
        g.out_pitch = lay.ap;
        g.out_plane = lay.a_plane;
        g.depth = lay.n;
        g.out = am;
        if ((rc = launch_gemm<kGram>(xmap[k & 1], xmap[k & 1], g, sms, s))) return rc;
        g.depth = lay.m;
        g.a = am;
        g.out = pm;
        if ((rc = launch_gemm<kPoly>(amap, amap, g, sms, s))) return rc;
        g.cols = lay.n;
        if (k + 1 < steps) {
            g.out = x[(k + 1) & 1];
            g.out_pitch = lay.xp;
            g.out_plane = lay.x_plane;
            if ((rc = launch_gemm<kApply>(pmap, xright[k & 1], g, sms, s))) return rc;
        } else {
            out.batch = batch;
            out.rows = lay.m;
            out.cols = lay.n;
            out.depth = lay.m;
            out.transposed = prep.transposed;
            if ((rc = launch_gemm<kResult>(pmap, xright[k & 1], out, sms, s))) return rc;
        }
    }
    return CIMEKV_OK;
}

bool valid_type(int t) { return t == CIMEKV_F32 || t == CIMEKV_BF16 || t == CIMEKV_F16; }

}  // namespace

extern "C" size_t cimekv_orthogonalize_workspace_bytes(int batch, int rows, int cols) {
    if (batch <= 0 || rows <= 0 || cols <= 0 || rows > kMaxSide || cols > kMaxSide || batch > 65535) return 0;
    return Layout(batch, rows, cols).bytes;
}

extern "C" int cimekv_orthogonalize(const void* g, int type, long long batch_stride, long long row_stride, int batch,
                                    int rows, int cols, int steps, float a, float b, float c, float eps, void* out,
                                    void* workspace, size_t workspace_bytes, void* stream) {
    NvtxRange nvtx_range("cimekv_orthogonalize");
    int rc = cimekv_internal_begin_call();
    if (rc || (rc = check_iteration(batch, rows, cols, steps, a, b, c, eps))) return rc;
    if (!valid_type(type)) return fail(CIMEKV_EINVAL_SHAPE, "unknown element type");
    if (batch == 0 || rows == 0 || cols == 0) return CIMEKV_OK;
    if (!g || !out) return fail(CIMEKV_EINVAL_SHAPE, "null pointer");
    if (batch_stride < 0 || row_stride < 0) return fail(CIMEKV_EINVAL_SHAPE, "negative stride");
    if (!workspace || workspace_bytes < Layout(batch, rows, cols).bytes)
        return fail(CIMEKV_EWORKSPACE, "orthogonalize workspace too small");
    if ((uintptr_t)workspace % 256) return fail(CIMEKV_EINVAL_SHAPE, "workspace must be 256-byte aligned");
    PrepParams prep = {};
    prep.g.base = g;
    prep.g.batch_stride = batch_stride;
    prep.g.row_stride = row_stride;
    prep.g.type = type;
    prep.eps = eps;
    GemmParams last = {};
    last.dst.base = out;
    last.dst.batch_stride = (long long)rows * cols;
    last.dst.type = type;
    return run(prep, last, batch, rows, cols, steps, a, b, c, static_cast<uint8_t*>(workspace), (cudaStream_t)stream);
}

extern "C" int cimekv_muon_step(int count, void* const* params, const void* const* grads, float* const* momenta,
                                int p_type, int g_type, int rows, int cols, float lr, const float* lr_device,
                                float momentum, int nesterov, float weight_decay, float scale, int steps, float a,
                                float b, float c, float eps, void* workspace, size_t workspace_bytes, void* stream) {
    NvtxRange nvtx_range("cimekv_muon_step");
    int rc = cimekv_internal_begin_call();
    if (rc || (rc = check_iteration(count, rows, cols, steps, a, b, c, eps))) return rc;
    if (count > kMaxTable) return fail(CIMEKV_EINVAL_SHAPE, "muon step: too many matrices for one call");
    if (!valid_type(p_type) || !valid_type(g_type)) return fail(CIMEKV_EINVAL_SHAPE, "unknown element type");
    if (!(momentum >= 0.0f && momentum <= 1.0f)) return fail(CIMEKV_EINVAL_SHAPE, "momentum must be in [0, 1]");
    if (count == 0 || rows == 0 || cols == 0) return CIMEKV_OK;
    if (!params || !grads || !momenta) return fail(CIMEKV_EINVAL_SHAPE, "null pointer");
    for (int i = 0; i < count; ++i)
        if (!params[i] || !grads[i] || !momenta[i]) return fail(CIMEKV_EINVAL_SHAPE, "null pointer");
    // matrices written in one launch must not share memory
    std::pair<uintptr_t, uintptr_t> range[2 * kMaxTable];
    const uintptr_t elements = (uintptr_t)rows * (uintptr_t)cols;
    for (int i = 0; i < count; ++i) {
        range[2 * i] = {(uintptr_t)params[i], (uintptr_t)params[i] + elements * (p_type == CIMEKV_F32 ? 4 : 2)};
        range[2 * i + 1] = {(uintptr_t)momenta[i], (uintptr_t)momenta[i] + elements * 4};
    }
    std::sort(range, range + 2 * count);
    for (int i = 1; i < 2 * count; ++i)
        if (range[i].first < range[i - 1].second)
            return fail(CIMEKV_EINVAL_SHAPE, "muon step: parameters and momenta must not overlap");
    if (!workspace || workspace_bytes < Layout(count, rows, cols).bytes)
        return fail(CIMEKV_EWORKSPACE, "muon step workspace too small");
    if ((uintptr_t)workspace % 256) return fail(CIMEKV_EINVAL_SHAPE, "workspace must be 256-byte aligned");
    PrepParams prep = {};
    GemmParams last = {};
    prep.g.tabled = prep.mom.tabled = last.dst.tabled = 1;
    prep.g.type = g_type;
    prep.mom.type = CIMEKV_F32;
    last.dst.type = p_type;
    prep.g.row_stride = cols;
    for (int i = 0; i < count; ++i) {
        prep.g.table[i] = const_cast<void*>(grads[i]);
        prep.mom.table[i] = momenta[i];
        last.dst.table[i] = params[i];
    }
    prep.beta = momentum;
    prep.nesterov = nesterov;
    prep.eps = eps;
    last.update = 1;
    last.lr = lr;
    last.lr_dev = lr_device;
    last.decay = weight_decay;
    last.scale = scale;
    return run(prep, last, count, rows, cols, steps, a, b, c, static_cast<uint8_t*>(workspace), (cudaStream_t)stream);
}
