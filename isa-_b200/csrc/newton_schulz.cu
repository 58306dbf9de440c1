// newton_schulz.cu — orthogonalisation of update matrices by Newton-Schulz
// products on the tensor cores, and the Muon optimiser step around it.
//
// With X0 = G / max(|G|_F, eps), m rows and n >= m columns (a tall G is worked on
// transposed), each step is
//
//   A = X X^T,   P = a I + b A + c A A,   X <- P X
//
// so the singular values s of X go through s (a + b s^2 + c s^4) and close in on
// one band around 1, while the singular vectors stay.  With the square completed,
//
//   B = X X^T + (b / 2c) I,   P = c B B + (a - b^2 / 4c) I,   X <- P X
//
// all three are one product each with an epilogue alpha D + beta I, so none of
// them reads anything but its operands.  For fp32 results of fewer than 224 rows P is formed as it
// stands, b A read by the second product's epilogue: the square's completion rounds A at
// the size of b / 2c (42 x 47: 1.7e-6 off, where products in fp32 are by 1.0e-6, and
// 1.0e-6 as it stands).  (c = 0: P = b X X^T + a I is the first product's, and the second falls away.)
//
// Precision.  A singular value far below the largest grows by up to a per step
// (x 485 in five steps), and so does any rounding noise in its direction: with
// operands rounded to 11 bits the result of a low-rank update is off by 1e-2, more
// than the half step of a bf16 result.  X, B and P are therefore held as pairs of
// fp16 planes, value * 2^12 = hi + lo.  Singular values stay below 15, checked on the host
// from the coefficients, so the fixed scale does not overflow.  Values from 2^-14 on keep 22 bits; below,
// where lo is subnormal, an element is off by up to 2^-37.  In norm that is 2^-37 sqrt(elements),
// 2^-23 of |X| = 1 for 16,384 x 16,384, no more than what 22 bits round off, and later steps only grow |X|.  A
// product is hi hi + hi lo + lo hi, accumulated in fp32 in tensor memory: three
// tensor core products.  fp32 results are off by 0.35 to 1.2 times what products in
// fp32 give (4096 x 4096 Gaussian to a few dominant directions in 42 x 47).
//
// B and P are symmetric: only tiles on and below the diagonal are computed, the
// epilogue stores each tile and its mirror image.

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <mutex>
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

int launched(const char* what) {
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) return CIMEKV_OK;
    char msg[256];
    snprintf(msg, sizeof(msg), "%s: %s", what, cudaGetErrorString(e));
    return fail(CIMEKV_ECUDA, msg);
}

constexpr float kScale = 4096.0f;  // fp16 planes hold value * 2^12
constexpr int kK = 64;             // depth of one stage: 64 halves = one 128-byte swizzle row
constexpr int kMaxStages = 6, kMaxBufs = 8;

// The three kinds of output tile (see product()), by their side, and how finely they sum.
template <int kSide, bool kFine>
struct Tile {
    static constexpr bool kPair = kSide == 256;
    static constexpr int kRanks = kPair ? 2 : 1;
    static constexpr int kRows = kSide / kRanks;            // rows of either operand that one CTA stages
    static constexpr int kStages = kSide == 64 ? 6 : 3;     // 192 KB of them
    static constexpr int kOperand = kRows * kK * 2;         // bytes of one operand plane in a stage
    static constexpr int kStageBytes = 4 * kOperand;        // left hi, left lo, right hi, right lo
    static constexpr int kWarpRows = kRows / 4;             // result rows of a collecting warp (its quarter of
                                                            // tensor memory; 64 rows fill half of each)
    static constexpr int kWarps = kSide == 64 ? 8 : 16;     // collecting warps
    static constexpr int kWarpCols = kSide / (kWarps / 4);  // result columns of a collecting warp
    static constexpr int kThreads = (kWarps + 2) * 32;      // and a copy warp, a product warp
    static constexpr int kBufs = kSide == 64 ? 8 : kPair ? 2 : 4;   // accumulators in tensor memory
    // Steps of 16 along K summed in one of them: half a stage or (fast) a stage, of a pair a
    // stage or (fast) two; the parts of a stage, and the stages, that this makes.
    static constexpr int kSums = (kPair ? 4 : 2) * (kFine ? 1 : 2);
    static constexpr int kParts = kSums < 4 ? 4 / kSums : 1, kSpan = kSums > 4 ? kSums / 4 : 1;
    static constexpr int kColumns = 512;                    // tensor memory columns taken: all
    static constexpr int kStaging = kWarpRows * 64;         // a collecting warp's row segments on their way out
    static constexpr int smem() { return kStages * kStageBytes + kWarps * kStaging + 1024; }
};

constexpr int kMaxTable = CIMEKV_MUON_MAX_MATRICES;
constexpr int kMaxParts = 512;              // partial norms per matrix, at most

// ------------------------------------------------------------- PTX pieces --

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

// Address of the same shared variable in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
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

// A warp's box of 32 columns from its staging place to a plane, and the wait until
// the place may be written again (all: until the planes are written).
__device__ __forceinline__ void tma_store(const CUtensorMap* map, uint32_t src, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];\n\t"
        "cp.async.bulk.commit_group;" ::"l"(map), "r"(src), "r"(x), "r"(y), "r"(z)
        : "memory");
}
template <bool kAll>
__device__ __forceinline__ void tma_store_wait() {
    if constexpr (kAll) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    else asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}

// One lane of a converged warp.  The copy and product warps run whole, with values
// that are the same in all lanes, and only issue from one: coordinates and
// descriptors then live in uniform registers, where these instructions want them
// (issued from an `if (lane == 0)` a stage's twelve products took 1,450 cycles).
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
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

// 16 accumulator columns of this lane's row.
__device__ __forceinline__ void tmem_load16(uint32_t addr, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
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
    float beta, gain;   // of the momentum and of the gradient
    int nesterov;
    int rows, cols;     // of G
    int transposed;     // rows > cols
    int pitch;          // of the planes, elements
    long long plane;    // elements from the hi to the lo plane
    float eps;
    int parts;          // partial norms per matrix
    double* part;       // [batch][parts]
    unsigned* arrivals; // [batch], zeroed here for ns_steps_kernel
    __half* x;
};

// The next kernel of the chain may be set up while this one runs, and this one
// touches memory only after the one before has finished and its writes are seen.
__device__ __forceinline__ void chain() {
    asm volatile("griddepcontrol.launch_dependents;\n\tgriddepcontrol.wait;" ::: "memory");
}

// The update before orthogonalisation: G itself, or the (Nesterov) momentum after
// its own update m <- beta m + gain g.
__device__ __forceinline__ float new_momentum(const PrepParams& p, float g, float m) { return fmaf(p.beta, m, p.gain * g); }
__device__ __forceinline__ float update_of(const PrepParams& p, float g, float m) {
    return p.nesterov ? fmaf(p.beta, m, p.gain * g) : m;
}

// Four neighbours from an address that is a multiple of four elements.
__device__ __forceinline__ void load4(const void* p, int type, long long i, float (&v)[4]) {
    if (type == CIMEKV_F32) {
        const float4 q = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
        v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else {
        const uint2 q = *reinterpret_cast<const uint2*>(static_cast<const unsigned short*>(p) + i);
        if (type == CIMEKV_BF16) {
            v[0] = __uint_as_float(q.x << 16); v[1] = __uint_as_float(q.x & 0xffff0000u);
            v[2] = __uint_as_float(q.y << 16); v[3] = __uint_as_float(q.y & 0xffff0000u);
        } else {
            const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&q.x));
            const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&q.y));
            v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
        }
    }
}

// Momentum update and the partial sums of squares of one matrix, p.parts CTAs
// to a matrix, in doubles (squares of fp32 values neither overflow nor vanish),
// added in a fixed order.  kFlat: a matrix is one run of elements that vectors of
// four fit; otherwise row by row.  Bound by HBM: 52 us for a Muon step's 48 of 768 x 768
// (340 MB in fp32, 6.5 TB/s), 22 to 27 us for 4,096 x 4,096 bf16, whose 33 MB are latency.
template <bool kFlat>
__global__ void __launch_bounds__(256) ns_norm_kernel(const __grid_constant__ PrepParams p) {
    const int b = blockIdx.y;
    const void* g = p.g.at(b);
    float* mom = p.mom.tabled ? static_cast<float*>(p.mom.table[b]) : nullptr;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (blockIdx.x == 0 && threadIdx.x == 0) p.arrivals[b] = 0;
    double s = 0.0;
    if constexpr (kFlat) {
        constexpr int kAhead = 4;
        const long long total = (long long)p.rows * p.cols / 4, step = (long long)p.parts * 256;
        for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += kAhead * step) {
            // loads of several turns first: one after the other they are latency
            float v[kAhead][4];
            float4 m[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                if (i + u * step < total) {
                    load4(g, p.g.type, 4 * (i + u * step), v[u]);
                    if (mom) m[u] = *reinterpret_cast<const float4*>(mom + 4 * (i + u * step));
                }
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                if (i + u * step >= total) break;
                if (mom) {
                    m[u].x = new_momentum(p, v[u][0], m[u].x);
                    m[u].y = new_momentum(p, v[u][1], m[u].y);
                    m[u].z = new_momentum(p, v[u][2], m[u].z);
                    m[u].w = new_momentum(p, v[u][3], m[u].w);
                    *reinterpret_cast<float4*>(mom + 4 * (i + u * step)) = m[u];
                    v[u][0] = update_of(p, v[u][0], m[u].x);
                    v[u][1] = update_of(p, v[u][1], m[u].y);
                    v[u][2] = update_of(p, v[u][2], m[u].z);
                    v[u][3] = update_of(p, v[u][3], m[u].w);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) s += (double)v[u][k] * (double)v[u][k];
            }
        }
    } else {
        for (int r = blockIdx.x; r < p.rows; r += p.parts)
            for (int c = threadIdx.x; c < p.cols; c += 256) {
                float v = load_as_float(g, p.g.type, r * p.g.row_stride + c);
                if (mom) {
                    const long long i = (long long)r * p.cols + c;
                    const float m = new_momentum(p, v, mom[i]);
                    mom[i] = m;
                    v = update_of(p, v, m);
                }
                s += (double)v * (double)v;
            }
    }
    __shared__ double red[8];
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; ++w) s += red[w];
        p.part[(long long)b * p.parts + blockIdx.x] = s;
    }
}

// The planes' words of two neighbours (packed conversions: one instruction for both).
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 back = __half22float2(h);
    const __half2 l = __floats2half2_rn(a - back.x, b - back.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}
// Two neighbours in a 16-bit type.
__device__ __forceinline__ uint32_t pack2(int type, float a, float b) {
    if (type == CIMEKV_BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// 2^12 / max(norm, eps) of matrix b, by the first warp for the whole CTA.
__device__ __forceinline__ float plane_factor(const PrepParams& p, int b, float* shared) {
    if (threadIdx.x < 32) {
        double s = 0.0;
        for (int i = threadIdx.x; i < p.parts; i += 32) s += p.part[(long long)b * p.parts + i];
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        const double norm = sqrt(s);
        if (threadIdx.x == 0)
            *shared = (float)((double)kScale / (norm > (double)p.eps || norm != norm ? norm : (double)p.eps));
    }
    __syncthreads();
    return *shared;
}

// X0 as pairs of planes: a thread's eight neighbours of one row (8 x 256 tiles).
// kVec: rows of G and of the momenta can be read in vectors of four.  Bound by HBM: 56 to 63 us
// for 48 of 768 x 768 with momenta (340 MB).
template <bool kVec>
__global__ void __launch_bounds__(256) ns_prepare_kernel(const __grid_constant__ PrepParams p) {
    __shared__ float shared;
    chain();
    // from the end: what ns_norm_kernel touched last is still in L2
    const int b = gridDim.z - 1 - blockIdx.z;
    const float factor = plane_factor(p, b, &shared);
    const int r = (gridDim.y - 1 - blockIdx.y) * 8 + (threadIdx.x >> 5), c = blockIdx.x * 256 + (threadIdx.x & 31) * 8;
    if (r >= p.rows || c >= p.cols) return;
    const void* g = p.g.at(b);
    const float* mom = p.mom.tabled ? static_cast<const float*>(p.mom.table[b]) + (long long)r * p.cols : nullptr;
    float v[8] = {};
    if constexpr (kVec) {
#pragma unroll
        for (int h = 0; h < 8; h += 4) {
            if (c + h < p.cols) {
                float q[4];
                load4(g, p.g.type, r * p.g.row_stride + c + h, q);
                if (mom) {
                    const float4 m = *reinterpret_cast<const float4*>(mom + c + h);
                    q[0] = update_of(p, q[0], m.x);
                    q[1] = update_of(p, q[1], m.y);
                    q[2] = update_of(p, q[2], m.z);
                    q[3] = update_of(p, q[3], m.w);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) v[h + k] = q[k];
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (c + k < p.cols) {
                v[k] = load_as_float(g, p.g.type, r * p.g.row_stride + c + k);
                if (mom) v[k] = update_of(p, v[k], mom[c + k]);
            }
    }
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) split2(v[2 * k] * factor, v[2 * k + 1] * factor, hi[k], lo[k]);
    // the pitch is a multiple of 8: a group that begins inside a row ends inside its pitch
    __half* x = p.x + ((long long)b * p.rows + r) * p.pitch + c;
    *reinterpret_cast<uint4*>(x) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    *reinterpret_cast<uint4*>(x + p.plane) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
}

// The same for a tall G, transposed: 64 x 64 tiles through shared memory, so
// that reads and writes are both along rows.
__global__ void __launch_bounds__(256) ns_prepare_tall_kernel(const __grid_constant__ PrepParams p) {
    __shared__ float tile[64][65];
    __shared__ float shared;
    chain();
    const int b = gridDim.z - 1 - blockIdx.z;
    const float factor = plane_factor(p, b, &shared);
    const void* g = p.g.at(b);
    const float* mom = p.mom.tabled ? static_cast<const float*>(p.mom.table[b]) : nullptr;
    const int r0 = (gridDim.y - 1 - blockIdx.y) * 64, c0 = blockIdx.x * 64;
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
#pragma unroll 4
    for (int k = ty; k < 64; k += 4) {
        const int r = r0 + k, c = c0 + tx;
        float v = 0.0f;
        if (r < p.rows && c < p.cols) {
            v = load_as_float(g, p.g.type, r * p.g.row_stride + c);
            if (mom) v = update_of(p, v, mom[(long long)r * p.cols + c]);
        }
        tile[k][tx] = v * factor;
    }
    __syncthreads();
    // X has cols rows and rows columns
    for (int i = threadIdx.x; i < 64 * 8; i += 256) {
        const int xr = i >> 3, k = (i & 7) * 8;
        if (c0 + xr >= p.cols || r0 + k >= p.rows) continue;
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) split2(tile[k + 2 * j][xr], tile[k + 2 * j + 1][xr], hi[j], lo[j]);
        __half* x = p.x + ((long long)b * p.cols + c0 + xr) * p.pitch + r0 + k;
        *reinterpret_cast<uint4*>(x) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(x + p.plane) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
}

// ---------------------------------------------------------------- products --

// kSymmetric: alpha L L^T + beta I, one triangle and its mirror image; kFull: the same, all
// tiles; kApply: L R; kResult: L R to the caller's matrices.
// kAny: one of the others, told at run time (all but kSymmetric).
enum Mode { kSymmetric = 0, kFull = 1, kApply = 2, kResult = 3, kAny = 4 };

// One product of a batch.
struct Product {
    int rows, cols, depth;
    float alpha, beta;      // on values as the planes hold them
    const __half* add;      // planes of which gamma times the value is added to the sum, or null (fine sums of
                            // ns_steps_kernel and 128 x 128 tiles only)
    long long add_plane;
    int add_pitch;
    float gamma;
};

// Where the last product goes.
struct Result {
    int transposed;
    int vec;                // rows of dst can be moved in vectors of 16 bytes
    Matrices dst;           // results, or parameters to update in place
    int update;             // parameters: p <- p (1 - lr decay) - lr scale X
    float lr, decay, scale;
    const float* lr_dev;
    unsigned* lost;         // marked when a wait has run out (by any product, not the last alone)
};

// Tile (i, j) of the lower triangle, row by row.
__device__ __forceinline__ void triangle(int t, int& i, int& j) {
    i = (int)((sqrtf(8.0f * (float)t + 1.0f) - 1.0f) * 0.5f);
    while ((i + 1) * (i + 2) / 2 <= t) ++i;
    while (i * (i + 1) / 2 > t) --i;
    j = t - i * (i + 1) / 2;
}

// The new value of an element of the result or parameter.
__device__ __forceinline__ float result_of(const Result& p, float sum, float old, float lr) {
    const float o = sum * (1.0f / (kScale * kScale));
    return p.update ? fmaf(-lr * p.scale, o, fmaf(-lr * p.decay, old, old)) : o;
}

// Turns rows held by lanes into row segments: on entry lane i < kRows holds 64 bytes
// of row i, on exit d[t] is bytes 16 (i % 4) .. + 15 of row 8 t + i / 4, so that a
// store covers eight segments of 64 bytes instead of 32 of 16 (an SM moves one
// 128-byte line a cycle however little of it is used: straight from the registers the
// stores of a 128 x 128 tile took 6,000 cycles).  Units of 16 bytes are
// swizzled: both sides are free of bank conflicts.
template <int kRows>
__device__ __forceinline__ void turn_rows(uint32_t staging, const uint4 (&r)[4], uint4 (&d)[kRows / 8]) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
    if (kRows == 32 || lane < kRows) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t at = staging + lane * 64 + ((k ^ ((lane >> 1) & 3)) << 4);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(r[k].x), "r"(r[k].y), "r"(r[k].z),
                         "r"(r[k].w)
                         : "memory");
        }
    }
    __syncwarp();
#pragma unroll
    for (int t = 0; t < kRows / 8; ++t) {
        const int row = 8 * t + (lane >> 2);
        const uint32_t at = staging + row * 64 + (((lane & 3) ^ ((row >> 1) & 3)) << 4);
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(d[t].x), "=r"(d[t].y), "=r"(d[t].z), "=r"(d[t].w)
                     : "r"(at)
                     : "memory");
    }
}

// 16 columns from cb of the warp's kRows rows from row0 of the last product, to the
// caller's matrix.  Called by whole warps.
template <int kRows>
__device__ __forceinline__ void finish_result(const Result& p, int rows, int cols, const float (&v)[16], int b, int row0,
                                              int cb, float lr, uint32_t staging) {
    void* dst = const_cast<void*>(p.dst.at(b));
    const int type = p.dst.type, lane = threadIdx.x & 31;
    if (p.transposed) {  // neighbouring lanes hold neighbouring elements
        const int r = row0 + lane;
        if (lane >= kRows || r >= rows) return;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (cb + i >= cols) break;
            const long long at = (long long)(cb + i) * rows + r;
            store_float(dst, type, at, result_of(p, v[i], p.update ? load_as_float(dst, type, at) : 0.0f, lr));
        }
        return;
    }
    uint4 in[4], out[kRows / 8];
#pragma unroll
    for (int k = 0; k < 4; ++k)
        in[k] = make_uint4(__float_as_uint(v[4 * k]), __float_as_uint(v[4 * k + 1]), __float_as_uint(v[4 * k + 2]),
                           __float_as_uint(v[4 * k + 3]));
    turn_rows<kRows>(staging, in, out);
    const int c = cb + (lane & 3) * 4;
#pragma unroll
    for (int t = 0; t < kRows / 8; ++t) {
        const int r = row0 + 8 * t + (lane >> 2);
        if (r >= rows || c >= cols) continue;
        const long long at = (long long)r * cols + c;
        const float x[4] = {__uint_as_float(out[t].x), __uint_as_float(out[t].y), __uint_as_float(out[t].z),
                            __uint_as_float(out[t].w)};
        if (p.vec) {  // rows of whole vectors
            float o[4] = {};
            if (p.update) load4(dst, type, at, o);
#pragma unroll
            for (int k = 0; k < 4; ++k) o[k] = result_of(p, x[k], o[k], lr);
            if (type == CIMEKV_F32) {
                *reinterpret_cast<float4*>(static_cast<float*>(dst) + at) = make_float4(o[0], o[1], o[2], o[3]);
            } else {
                uint32_t q[2];
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    q[k] = pack2(type, o[2 * k], o[2 * k + 1]);
                *reinterpret_cast<uint2*>(static_cast<unsigned short*>(dst) + at) = make_uint2(q[0], q[1]);
            }
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (c + k < cols)
                    store_float(dst, type, at + k,
                                result_of(p, x[k], p.update ? load_as_float(dst, type, at + k) : 0.0f, lr));
        }
    }
}

// 32 columns from cb of a lane's row of the planes that a product adds to.
struct Addend {
    uint4 plane[2][4];
};
template <int kRows>
__device__ __forceinline__ void load_addend(const Product& p, int b, int row0, int cb, Addend& more) {
    const int lane = threadIdx.x & 31, r = row0 + lane;
    if (lane >= kRows || r >= p.rows) return;
    const __half* at = p.add + ((long long)b * p.rows + r) * p.add_pitch + cb;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        if (cb + 8 * q >= p.cols) break;
#pragma unroll
        for (int i = 0; i < 2; ++i)  // written by other SMs while this kernel runs: not from L1
            more.plane[i][q] = __ldcg(reinterpret_cast<const uint4*>(at + i * p.add_plane + 8 * q));
    }
}

__device__ __forceinline__ void add_addend(float gamma, const Addend& more, float (&v0)[16], float (&v1)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const auto word = [&](const uint4& u) { return i % 4 == 0 ? u.x : i % 4 == 1 ? u.y : i % 4 == 2 ? u.z : u.w; };
        const uint32_t wh = word(more.plane[0][i / 4]), wl = word(more.plane[1][i / 4]);
        const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&wh));
        const float2 l = __half22float2(*reinterpret_cast<const __half2*>(&wl));
        float* v = i < 8 ? &v0[2 * i] : &v1[2 * i - 16];
        v[0] = fmaf(gamma, h.x + l.x, v[0]);
        v[1] = fmaf(gamma, h.y + l.y, v[1]);
    }
}

// 32 columns from cb of the warp's kRows rows from row0 of a product that stays in
// planes (`diagonal`: a tile on the diagonal, which gets beta there; kMirror: off it,
// their mirror image too).  Rows of 64 bytes are staged in the 64-byte swizzle of `out` and leave by a
// bulk copy, which clips them to the matrix and lets the warp go on: ordinary stores of
// a 256 x 256 tile took 8,000 cycles, in which the products ran out of accumulators.
// Called by whole warps.
template <bool kMirror, int kRows>
__device__ __forceinline__ void finish_planes(const Product& p, const CUtensorMap* out, const float (&v0)[16],
                                              const float (&v1)[16], int batch, int b, int row0, int cb, bool diagonal,
                                              uint32_t staging) {
    const int lane = threadIdx.x & 31, r = row0 + lane;
    uint32_t words[2][16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float o[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            o[k] = (i < 8 ? v0[(2 * i + k) & 15] : v1[(2 * i + k) & 15]) * p.alpha;
            if (diagonal && r == cb + 2 * i + k) o[k] += p.beta;
        }
        split2(o[0], o[1], words[0][i], words[1][i]);
    }
    const auto leave = [&](int x, int y, int plane) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) tma_store(out, staging, x, y, plane * batch + b);
    };
    const auto place_free = [&]() {
        if (lane == 0) tma_store_wait<false>();
        __syncwarp();
    };
    if (row0 >= p.rows) return;
#pragma unroll
    for (int plane = 0; plane < 2; ++plane) {
        const uint32_t(&w)[16] = words[plane];
        place_free();
        if (kRows == 32 || lane < kRows) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t at = staging + lane * 64 + ((k ^ ((lane >> 1) & 3)) << 4);
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[4 * k]), "r"(w[4 * k + 1]),
                             "r"(w[4 * k + 2]), "r"(w[4 * k + 3])
                             : "memory");
            }
        }
        leave(cb, row0, plane);
        if (kMirror && !diagonal) {  // row c of the image: element c of all lanes
            place_free();
#pragma unroll
            for (int c = 0; c < 32; ++c) {
                const uint32_t at = staging + c * 64 + (((lane >> 3) ^ ((c >> 1) & 3)) << 4) + (lane & 7) * 2;
                asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"((unsigned short)(w[c / 2] >> (16 * (c & 1)))) : "memory");
            }
            leave(row0, cb, plane);
        }
    }
}

// Place in a ring of barriers and the parity of the phase to wait for there.  (Kept
// step by step: the divisions of a running number were 250 cycles a stage in the one
// thread that issues.)
struct Turn {
    int at;
    uint32_t parity;
    __device__ __forceinline__ void next(int places) {
        if (++at == places) {
            at = 0;
            parity ^= 1;
        }
    }
};

// Shared-memory addresses of a CTA's pipeline, and where each role stands in it.
struct Pipe {
    uint32_t stages, full, empty, acc_full, acc_empty, tmem;
    uint32_t rank;          // in the pair
    Turn fill;              // copy and product warps: the stage
    Turn chunk;             // product and collecting warps: the accumulator
    bool ok;                // no wait has run out
};

// Where the CTAs of a matrix meet between the products of ns_steps_kernel: a
// collecting warp counts itself in when its part of the result is in memory, and
// only what depends on the others waits: the copy warp, before it asks for their results.
struct Meet {
    unsigned* arrivals;     // of the matrix, zeroed by ns_norm_kernel
    unsigned target;        // CTAs' arrivals until the last product's end; 0: nothing to wait for
    uint32_t own;           // barrier of a CTA that has a matrix alone; 0: it has not
    uint32_t counted;       // warps of the CTA that have counted themselves in; the last one counts for all
    volatile int* lost;     // set when a wait has run out: from then on none is waited for and all results are NaN
    unsigned* word;         // and what tells the host
};
template <int kWarps>
__device__ __forceinline__ void meet_arrive(const Meet& m) {
    asm volatile("fence.proxy.async.global;" ::: "memory");  // planes are written and read by copies
    if (m.own) {
        asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(m.own) : "memory");
        return;
    }
    unsigned before;
    asm volatile("atom.acq_rel.cta.shared::cta.add.u32 %0, [%1], 1;" : "=r"(before) : "r"(m.counted) : "memory");
    if (before % kWarps == kWarps - 1) asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(m.arrivals) : "memory");
}
// Called by whole warps.  For two seconds at most.
__device__ __forceinline__ void meet_wait(const Meet& m) {
    bool ok = true;
    if (*m.lost) return;
    if (m.target && m.own) {
        ok = mbar_wait(m.own, (m.target - 1) & 1);
    } else if (m.target) {
        Patience patience;
        for (;;) {
            unsigned seen;
            asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(m.arrivals) : "memory");
            if (seen >= m.target) break;
            if (!patience.left()) {
                ok = false;
                break;
            }
        }
    }
    if (!ok) {
        *m.lost = 1;
        __threadfence_block();
        mark_lost(m.word);
    }
    asm volatile("fence.proxy.async.global;" ::: "memory");
    __syncwarp();
}

// The tiles first, first + step, ... of one product: of matrix `matrix`, or (-1) of all
// matrices in turn.  Tiles are 128 x 128 by one CTA,
// 256 x 256 by a pair of CTAs whose tensor cores work as one (each stages 128
// rows of either operand, holds its 128 rows of the result, and the first CTA
// issues), or 64 x 64 by one CTA.  One warp copies stages ahead, one
// issues products, the others collect.  An SM takes in about 43 bytes a cycle and
// puts out about 30: a stage of 64 KB (768 cycles of products for a 128 tile, 1,536
// for a pair) feeds only the pair's tensor cores, which is why many tiles go to
// pairs and few to the tile that spreads them over the most SMs.
//
// The tensor core aligns the 16 products of a step and the accumulator to the largest
// of them and cuts off below about 2^-25 of it (a model of that on the CPU gives
// the errors that are measured), so errors grow with what is already summed and all
// have one sign.  So a few steps (the small cross products before those at full size) go
// into a fresh accumulator, one of several, and the collecting warps add them in
// registers with round-to-nearest while the next ones run.  With the square completed 192 x 192 is off
// by 1.8e-6 with fine sums (products in fp32 1.6e-6, coarse sums 2.8e-6), 48 of 768 x 768 by 2.6e-6 (2.4e-6,
// 4.6e-6).  Fine sums take 40 of 192 x 192 146 us instead of 125 in the one kernel (a Muon step each); where the products
// are kernels the power limit hides them.  The same accumulators let the next tile start while the last one is stored.
template <int M, int kSide, bool kFine>
__device__ __forceinline__ void product(Pipe& q, const CUtensorMap* left, const CUtensorMap* right,
                                        const CUtensorMap* out, const Product& p, const Result& result, int batch, int first, int step, int tiles,
                                        int mode = M, int matrix = -1, const Meet& meet = Meet()) {
    using T = Tile<kSide, kFine>;
    constexpr bool kPair = T::kPair;
    constexpr int kRanks = T::kRanks, kRows = T::kRows, kOperand = T::kOperand, kStageBytes = T::kStageBytes;
    constexpr int kWarpCols = T::kWarpCols, kWarps = T::kWarps, kBufs = T::kBufs;
    constexpr int kStages = T::kStages;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // known to be uniform
    const int ni = (p.rows + kSide - 1) / kSide, nj = (p.cols + kSide - 1) / kSide;
    const int per_matrix = M == kSymmetric ? ni * (ni + 1) / 2 : ni * nj;
    const int ksteps = (p.depth + kK - 1) / kK;
    const bool square = mode <= kFull;  // L L^T: both operands' rows run along K
    const float per_row = 1.0f / (float)nj;
    const auto place = [&](int t, int& b, int& row0, int& col0) {
        b = matrix >= 0 ? matrix : t / per_matrix;
        const int at = matrix >= 0 ? t : t - b * per_matrix;
        int i, j;
        if (M == kSymmetric) {
            triangle(at, i, j);
        } else {
            i = (int)((float)at * per_row);  // off by one at most (at < 2^24), mended below
            j = at - i * nj;
            if (j < 0) {
                --i;
                j += nj;
            } else if (j >= nj) {
                ++i;
                j -= nj;
            }
        }
        row0 = i * kSide;
        col0 = j * kSide;
    };

    if (warp == kWarps) {
        const uint32_t count_at = kPair ? cluster_addr(q.full, 0) : q.full;
        int ahead = 0;  // stages of the first tile that have their right operand on the way
        if constexpr (M == kAny) {
            if (!square && first < tiles) {  // X stands since the step before: it need not wait for the others
                int b, row0, col0;
                place(first, b, row0, col0);
                Turn fill = q.fill;
                for (; ahead < ksteps && ahead < kStages; ++ahead, fill.next(kStages)) {
                    if (!(q.ok = q.ok && mbar_wait(q.empty + 8 * fill.at, fill.parity ^ 1))) break;
                    if (elect_one()) {
                        mbar_expect(q.full + 8 * fill.at, kStageBytes);
#pragma unroll
                        for (int plane = 0; plane < 2; ++plane)
                            tma_box<kPair>(q.stages + fill.at * kStageBytes + (2 + plane) * kOperand, right, col0, ahead * kK,
                                           plane * batch + b, q.full + 8 * fill.at);
                    }
                    __syncwarp();
                }
            }
            meet_wait(meet);
        }
        for (int t = first; t < tiles && q.ok; t += step) {
            int b, row0, col0;
            place(t, b, row0, col0);
            const bool same = square && row0 == col0;  // both operands are the same rows
            row0 += (int)q.rank * kRows;
            col0 += (int)q.rank * kRows;
            for (int k = 0; k < ksteps; ++k, q.fill.next(kStages)) {
                const int s = q.fill.at;
                // (the phase before a barrier's first has ended by definition)
                const bool asked = M == kAny && t == first && k < ahead;
                if (!asked && !(q.ok = mbar_wait(q.empty + 8 * s, q.fill.parity ^ 1))) break;
                const uint32_t base = q.stages + s * kStageBytes, bar = count_at + 8 * s;
                if (elect_one()) {
                    if (q.rank == 0 && !asked) mbar_expect(q.full + 8 * s, kRanks * (same ? kStageBytes / 2 : kStageBytes));
#pragma unroll
                    for (int plane = 0; plane < 2; ++plane) {
                        const int z = plane * batch + b;
                        const uint32_t l = base + plane * kOperand, r = base + (2 + plane) * kOperand;
                        tma_box<kPair>(l, left, k * kK, row0, z, bar);
                        if (same || asked) continue;
                        if (square) {
                            tma_box<kPair>(r, right, k * kK, col0, z, bar);
                        } else {
                            tma_box<kPair>(r, right, col0, k * kK, z, bar);
                            if (kRows == 128) tma_box<kPair>(r + kOperand / 2, right, col0 + 64, k * kK, z, bar);
                        }
                    }
                }
                __syncwarp();
            }
        }
    } else if (warp == kWarps + 1) {
        if (q.rank == 0) {
            // D fp32, A and B fp16; right operand along K (0) or along its own axis (1)
            const uint32_t idesc = 1u << 4 | (square ? 0u : 1u << 16) | (uint32_t)(kSide / 8) << 17 |
                                   (uint32_t)(kSide / 16) << 24;
            for (int t = first; t < tiles && q.ok; t += step) {
                int b, row0, col0;
                place(t, b, row0, col0);
                const int r_at = square && row0 == col0 ? 0 : 2 * kOperand;  // on the diagonal L is R
                for (int k = 0; k < ksteps && q.ok; ++k, q.fill.next(kStages)) {
                    const int s = q.fill.at;
                    if (!(q.ok = mbar_wait(q.full + 8 * s, q.fill.parity))) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t base = q.stages + s * kStageBytes;
                    // both planes of either operand; a step of 16 along K moves the address alone
                    const uint64_t l0 = operand_desc(base, 16, 1024), l1 = operand_desc(base + kOperand, 16, 1024);
                    const uint64_t r0 = operand_desc(base + r_at, square ? 16 : 8192, 1024);
                    const uint64_t r1 = operand_desc(base + r_at + kOperand, square ? 16 : 8192, 1024);
                    const uint64_t kL = 32 >> 4, kR = (square ? 32 : 2048) >> 4;
                    constexpr int kHere = kK / 16 / T::kParts;  // steps of a part
                    const bool fresh = k % T::kSpan == 0, last = (k + 1) % T::kSpan == 0 || k + 1 == ksteps;
#pragma unroll
                    for (int part = 0; part < T::kParts; ++part) {
                        const int buf = q.chunk.at;
                        if (fresh && !(q.ok = mbar_wait(q.acc_empty + 8 * buf, q.chunk.parity ^ 1))) break;
                        const uint32_t d = q.tmem + buf * kSide;
                        if (elect_one()) {
#pragma unroll
                            for (uint64_t i = part * kHere; i < (part + 1) * kHere; ++i) {
                                mma_f16<kPair>(d, l0 + i * kL, r1 + i * kR, idesc, i != part * kHere || !fresh);
                                mma_f16<kPair>(d, l1 + i * kL, r0 + i * kR, idesc, 1);
                            }
#pragma unroll
                            for (uint64_t i = part * kHere; i < (part + 1) * kHere; ++i)
                                mma_f16<kPair>(d, l0 + i * kL, r0 + i * kR, idesc, 1);
                            if (last) mma_commit<kPair>(q.acc_full + 8 * buf);
                            if (part + 1 == T::kParts) mma_commit<kPair>(q.empty + 8 * s);
                        }
                        __syncwarp();
                        if (last) q.chunk.next(kBufs);
                    }
                }
            }
        }
    } else {
        const int quarter = warp & 3, group = warp >> 2;
        const uint32_t staging = q.stages + kStages * kStageBytes + warp * T::kStaging;
        const uint32_t empty_at = kPair ? cluster_addr(q.acc_empty, 0) : q.acc_empty;
        float lr = 0.0f;
        if (mode == kResult && result.update) lr = result.lr_dev ? *result.lr_dev : result.lr;
        for (int t = first; t < tiles; t += step) {
            int b, row0, col0;
            place(t, b, row0, col0);
            const int r0 = row0 + (int)q.rank * kRows + quarter * T::kWarpRows;
            const bool diagonal = square && row0 == col0;
            col0 += group * kWarpCols;
            float acc[kWarpCols / 16][16];
#pragma unroll
            for (int g = 0; g < kWarpCols / 16; ++g)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[g][i] = 0.0f;
            // a 64 x 64 tile's addend is asked for once its first sums are there (A stands by then) and
            // comes while the next ones run
            constexpr bool kAdd = kFine && (M == kAny || (M == kSymmetric && kSide == 128)), kEarly = kAdd && kSide == 64;
            Addend more = {};
            for (int k = 0; k < ksteps * (kK / 16); k += T::kSums, q.chunk.next(kBufs)) {
                const int buf = q.chunk.at;
                q.ok = q.ok && mbar_wait(q.acc_full + 8 * buf, q.chunk.parity);
                if (kEarly && k == 0 && p.add) load_addend<T::kWarpRows>(p, b, r0, col0, more);
                q.ok = __all_sync(0xffffffffu, q.ok);
                if (!q.ok) continue;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t src = q.tmem + ((uint32_t)(quarter * 32) << 16) + buf * kSide + group * kWarpCols;
#pragma unroll
                for (int g = 0; g < kWarpCols / 16; ++g) {
                    float v[16];
                    tmem_load16(src + g * 16, v);
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[g][i] += v[i];
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(empty_at + 8 * buf);
            }
            bool good = q.ok;
            if constexpr (M == kAny) good = __all_sync(0xffffffffu, good && !*meet.lost);
            if (!good) {  // a lost copy, product or meeting shows as NaN, it never passes for a result
#pragma unroll
                for (int g = 0; g < kWarpCols / 16; ++g)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[g][i] = __int_as_float(0x7fffffff);
            }
#pragma unroll
            for (int g = 0; g < kWarpCols / 16; ++g) {
                if (col0 + g * 16 >= p.cols) break;
                if (mode == kResult)
                    finish_result<T::kWarpRows>(result, p.rows, p.cols, acc[g], b, r0, col0 + g * 16, lr, staging);
                else if (g % 2 == 0) {
                    if (kAdd && p.add) {
                        if (!kEarly) load_addend<T::kWarpRows>(p, b, r0, col0 + g * 16, more);
                        add_addend(p.gamma, more, acc[g], acc[g + 1]);
                    }
                    finish_planes<M == kSymmetric, T::kWarpRows>(p, out, acc[g], acc[g + 1], batch, b, r0, col0 + g * 16,
                                                                 diagonal, staging);
                }
            }
            __syncwarp();
        }
        if (mode != kResult && lane == 0) tma_store_wait<true>();
        if (M == kAny && mode != kResult) {
            // without a tile nothing has held this warp back: its next arrival must not stand for another's last one
            if (first >= tiles) meet_wait(meet);
            if (lane == 0) meet_arrive<kWarps>(meet);
        }
        __syncwarp();
    }
}

// Barriers, tensor memory.  All threads.
template <typename T>
__device__ __forceinline__ void pipe_open(Pipe& q, uint64_t* bars, uint32_t* tmem_slot, uint8_t* smem_raw) {
    constexpr bool kPair = T::kPair;
    constexpr int kStages = T::kStages;
    q.stages = (smem_addr(smem_raw) + 1023) & ~1023u;
    q.full = smem_addr(bars);
    q.empty = q.full + 8 * kStages;
    q.acc_full = q.full + 16 * kStages;
    q.acc_empty = q.acc_full + 8 * kMaxBufs;
    q.rank = kPair ? cluster_rank() : 0;
    q.fill = q.chunk = {0, 0};
    q.ok = true;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(q.full + 8 * s, 1);
            mbar_init(q.empty + 8 * s, 1);
        }
        for (int s = 0; s < T::kBufs; ++s) {
            mbar_init(q.acc_full + 8 * s, 1);
            mbar_init(q.acc_empty + 8 * s, T::kWarps * T::kRanks);
        }
        mbar_init(q.acc_empty + 8 * kMaxBufs, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if ((threadIdx.x >> 5) == T::kWarps + 1) tmem_alloc<kPair>(smem_addr(tmem_slot), T::kColumns);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if constexpr (kPair) cluster_sync();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    q.tmem = *tmem_slot;
}

// Nothing may be in flight when the CTA leaves: copies (a pair's are all
// counted in the first CTA), products.  All threads.
template <typename T>
__device__ __forceinline__ void pipe_close(Pipe& q, unsigned* word) {
    if (!q.ok) mark_lost(word);
    constexpr bool kPair = T::kPair;
    constexpr int kWarps = T::kWarps, kStages = T::kStages;
    const int warp = threadIdx.x >> 5;
    if (warp == kWarps && q.rank == 0) {
        // a stage before the turn was last filled in this phase, the others in the one before
        for (int s = 0; s < kStages; ++s) mbar_wait(q.full + 8 * s, s < q.fill.at ? q.fill.parity : q.fill.parity ^ 1);
    } else if (warp == kWarps + 1 && q.rank == 0) {
        if (elect_one()) mma_commit<kPair>(q.acc_empty + 8 * kMaxBufs);
        __syncwarp();
        mbar_wait(q.acc_empty + 8 * kMaxBufs, 0);
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if constexpr (kPair) cluster_sync();  // the other CTA may still signal or read here
    if (warp == kWarps + 1) {
        __syncwarp();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        tmem_free<kPair>(q.tmem, T::kColumns);
    }
}

// One product of all matrices, a persistent loop over its tiles.  Counting the three
// tensor core products, on a GPU that was idle before: 4,096 x 4,096 in 281 to 299 us (P X) and 150 us (X X^T), 1,450
// TFLOP/s; 48 of 768 x 768 X X^T in 73 us at 1.8 GHz, 63 % of the tensor pipe: twelve stages a tile leave the intake
// of a tile's ends uncovered.  In a loop of calls the power limit takes the clock, and these are 105 (X X^T), 127
// (P X) and 200 us (the last product with the parameters' update, which reads and writes 226 MB).  The
// pair's kernels spill 28 to 140 bytes a thread outside the loop over the sums.
template <int M, int kSide, bool kFine>
__global__ void __launch_bounds__(Tile<kSide, kFine>::kThreads, 1) ns_gemm_kernel(const __grid_constant__ CUtensorMap left,
                                                                           const __grid_constant__ CUtensorMap right,
                                                                           const __grid_constant__ CUtensorMap out,
                                                                           const __grid_constant__ Product p,
                                                                           const __grid_constant__ Result result, int batch,
                                                                           int tiles) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[2 * kMaxStages + 2 * kMaxBufs + 1];
    __shared__ uint32_t tmem_slot;
    Pipe q;
    using T = Tile<kSide, kFine>;
    pipe_open<T>(q, bars, &tmem_slot, smem_raw);
    chain();
    constexpr int kRanks = T::kRanks;
    product<M, kSide, kFine>(q, &left, &right, &out, p, result, batch, blockIdx.x / kRanks, gridDim.x / kRanks, tiles);
    pipe_close<T>(q, result.lost);
}

// All steps in one kernel, for matrices whose products are a few microseconds
// each, less than it takes to end one kernel and start the next: `group` CTAs work on
// a matrix with 64 x 64 tiles and meet between its products.  A cooperative
// launch, so that all of them are resident while they wait for one another.
struct Steps {
    Product product[3];             // X X^T, its square, P X
    int squared;                    // 0: c = 0, no square
    unsigned* arrivals;             // per matrix, zeroed by ns_norm_kernel
    int steps, group;
};
struct StepMaps {
    CUtensorMap x[2], b, p;                 // to read from, boxes of 64 rows
    CUtensorMap x_out[2], b_out, p_out;     // to write to, boxes of a warp's rows
};

// All steps of matrices whose tiles fit the SMs, a group of CTAs to a matrix that meet
// after each product.  Bound by latency: a product of one 192 x 192 matrix is 63 us / 15 =
// 4.2 us (bf16; fp32 72 / 15 = 4.8), of which the meeting is about 1 us, the first copy 0.4, a stage 0.45 each (three),
// the way out 0.75.  This kernel alone, 16-bit results or a step's parameters / fp32 results: 40 of 192 x 192 in 110 / 142 us,
// 10 of 192 x 768 in 102 / 114, 2 of 257 x 1001 in 110.
template <bool kFine>
__global__ void __launch_bounds__(Tile<64, kFine>::kThreads, 1) ns_steps_kernel(const __grid_constant__ StepMaps maps,
                                                                         const __grid_constant__ Steps st,
                                                                         const __grid_constant__ Result result, int batch) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[2 * kMaxStages + 2 * kMaxBufs + 1];
    __shared__ __align__(8) uint64_t own;
    __shared__ int lost;
    __shared__ unsigned counted;
    __shared__ uint32_t tmem_slot;
    constexpr int kWarps = Tile<64, kFine>::kWarps;
    if (threadIdx.x == 0) {  // made known by pipe_open
        mbar_init(smem_addr(&own), kWarps);
        lost = 0;
        counted = 0;
    }
    Pipe q;
    pipe_open<Tile<64, kFine>>(q, bars, &tmem_slot, smem_raw);
    const int ni = (st.product[0].rows + 63) / 64, nj = (st.product[2].cols + 63) / 64;
    const int rank = blockIdx.x % st.group, groups = gridDim.x / st.group;
    Meet meet = {nullptr, 0, st.group > 1 ? 0 : smem_addr(&own), smem_addr(&counted), &lost, result.lost};
    unsigned met = 0;  // phases of `own` that earlier matrices have ended
    for (int matrix = blockIdx.x / st.group; matrix < batch; matrix += groups) {
        meet.arrivals = st.arrivals + matrix;
        unsigned count = 0;
        for (int k = 0; k < st.steps; ++k) {
            // All tiles of the square products: storing mirror images takes a CTA longer than a tile that
            // another one has time for.
            for (int i = 0; i < 3; i += st.squared ? 1 : 2) {
                const int mode = i < 2 ? kFull : k + 1 < st.steps ? kApply : kResult;
                const int tiles = ni * (i < 2 ? ni : nj);
                const CUtensorMap* const x = &maps.x[k & 1];
                product<kAny, 64, kFine>(q, i == 0 ? x : i == 1 ? &maps.b : &maps.p, i == 1 ? &maps.b : x,
                                  i == 0 && st.squared ? &maps.b_out : i < 2 ? &maps.p_out : &maps.x_out[(k + 1) & 1],
                                  st.product[i], result, batch, rank, st.group, tiles, mode, matrix, meet);
                if (mode != kResult) count += st.group;
                meet.target = count ? (meet.own ? met : 0) + count : 0;
            }
        }
        meet.target = 0;  // the next matrix begins with what ns_prepare_kernel left
        met += count;
    }
    pipe_close<Tile<64, kFine>>(q, result.lost);
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

// Planes [2 * batch][rows][cols] of a given pitch, zeros outside.
// To read: 64 columns, 128-byte swizzle; to write: 32 columns, 64-byte swizzle.
int plane_map(EncodeFn encode, CUtensorMap* map, __half* base, int batch, int rows, int cols, int pitch, int box_rows,
              bool write = false) {
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)2 * batch};
    const cuuint64_t strides[2] = {(cuuint64_t)pitch * 2, (cuuint64_t)pitch * 2 * rows};
    const cuuint32_t box[3] = {write ? 32u : 64u, (cuuint32_t)box_rows, 1}, step[3] = {1, 1, 1};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, base, dims, strides, box, step,
                              CU_TENSOR_MAP_INTERLEAVE_NONE,
                              write ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? CIMEKV_OK : fail(CIMEKV_ECUDA, "cuTensorMapEncodeTiled refused a plane");
}

// Workspace: partial norms, X twice, A, P (pairs of planes each).
struct Layout {
    int m, n, xp, ap;               // sides (m <= n) and pitches
    int parts;                      // partial norms per matrix: one per 4096 elements
    size_t part, arrivals, x0, x1, a, p, bytes;
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
        const long long want = ((long long)rows * cols + 4095) / 4096;
        parts = want < kMaxParts ? (int)want : kMaxParts;
        part = take((size_t)batch * parts * sizeof(double));
        arrivals = take((size_t)batch * sizeof(unsigned));
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
    const long long tiles = ((rows + 127LL) / 128) * ((cols + 127LL) / 128) * batch;
    if (tiles > 0x3fffffff) return fail(CIMEKV_EINVAL_SHAPE, "orthogonalize: too many elements for one call");
    if (steps < 1 || steps > 64) return fail(CIMEKV_EINVAL_SHAPE, "orthogonalize: 1 to 64 steps");
    // 2^12 / eps must be finite, or a matrix of zeros would give NaN
    if (!(eps >= 1e-30f)) return fail(CIMEKV_EINVAL_SHAPE, "eps must be at least 1e-30");
    if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c))
        return fail(CIMEKV_EINVAL_SHAPE, "orthogonalize: coefficients must be finite");
    // Largest singular values of X, B and P over the steps: they must fit the
    // planes' fixed scale (2^16 / 2^12).  For a singular value t of X, u = t^2, these are
    // t |p(u)|, |u + b / 2c| and |p(u)|, p(u) = a + b u + c u^2: largest at an end or where a derivative
    // vanishes (a + 3 b u + 5 c u^2 = 0, b + 2 c u = 0).  1 us for five steps.
    const double da = a, db = b, dc = c, shift = c != 0.0f ? 0.5 * db / dc : 0.0;
    double at[5] = {0.0, 0.0, 0.0, 0.0, 0.0};  // last: the end, s^2
    if (c != 0.0f) {
        const double d = 9.0 * db * db - 20.0 * da * dc;
        const double q = d >= 0.0 ? -0.5 * (3.0 * db + std::copysign(std::sqrt(d), db)) : 0.0;
        at[1] = q / (5.0 * dc);
        at[2] = q != 0.0 ? da / q : 0.0;
        at[3] = -shift;
    } else if (b != 0.0f) {
        at[1] = -da / (3.0 * db);
    }
    double s = 1.001;
    for (int k = 0; k < steps; ++k) {
        double next = 0.0, most = 0.0;
        at[4] = s * s;
        for (const double u : at) {
            if (!(u >= 0.0 && u <= at[4])) continue;
            const double p = std::fabs(da + (db + dc * u) * u);
            next = std::fmax(next, std::sqrt(u) * p);
            most = std::fmax(most, std::fmax(p, std::fabs(u + shift)));
        }
        s = next * 1.001;
        if (!(s <= 3.9 && most <= 15.0))
            return fail(CIMEKV_EINVAL_SHAPE,
                        "orthogonalize: these coefficients let singular values grow beyond 3.9, or a + b s^2 + c s^4 or "
                        "s^2 + b / 2c beyond 15");
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

// Lets `kernel` use its shared memory, once per device (the attribute stays).
template <typename Kernel>
int allow_smem(Kernel kernel, size_t bytes, std::atomic<uint64_t>& done) {
    int dev;
    if (cudaGetDevice(&dev) != cudaSuccess) return fail(CIMEKV_ECUDA, "no current device");
    if (dev < 64 && (done.load(std::memory_order_acquire) >> dev & 1)) return CIMEKV_OK;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e != cudaSuccess) return fail(CIMEKV_ECUDA, cudaGetErrorString(e));
    if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_release);
    return CIMEKV_OK;
}

long long tile_count(int mode, int side, int rows, int cols) {
    const long long ni = (rows + side - 1) / side, nj = (cols + side - 1) / side;
    return mode == kSymmetric ? ni * (ni + 1) / 2 : ni * nj;
}

// Launches `kernel` as a link of the chain (see chain()).
template <typename... Args>
int launch_chained(const char* what, void (*kernel)(Args...), dim3 grid, int threads, size_t smem, int cluster,
                   cudaStream_t s, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e == cudaSuccess) return CIMEKV_OK;
    (void)cudaGetLastError();
    char msg[256];
    snprintf(msg, sizeof(msg), "%s: %s", what, cudaGetErrorString(e));
    return fail(CIMEKV_ECUDA, msg);
}

template <int M, int kSide, bool kFine>
int launch_as(const CUtensorMap& l, const CUtensorMap& r, const CUtensorMap& out, const Product& p, const Result& result, int batch, int sms,
              cudaStream_t s) {
    using T = Tile<kSide, kFine>;
    static std::atomic<uint64_t> allowed{0};
    if (int rc = allow_smem(ns_gemm_kernel<M, kSide, kFine>, T::smem(), allowed)) return rc;
    constexpr int ranks = T::kRanks;
    const long long tiles = tile_count(M, kSide, p.rows, p.cols) * batch, most = sms / ranks;
    return launch_chained("ns_gemm_kernel", ns_gemm_kernel<M, kSide, kFine>, dim3((unsigned)(tiles < most ? tiles : most) * ranks),
                          T::kThreads, T::smem(), ranks, s, l, r, out, p, result, batch, (int)tiles);
}

// What a product takes, in cycles: a part that does not depend on its size (launch
// or meeting, latencies) and the tiles of the busiest SM, so many cycles a stage
// and a tile.  Fitted to times of single matrices of 64 to 1,280 rows and of
// batches of 8 to 200 matrices of 64 to 768 (within 15 %).
struct Cost {
    double start, stage, tile;
    double of(long long rounds, int depth) const { return start + rounds * (stage * ((depth + 63) / 64) + tile); }
};
constexpr Cost kCost64 = {5000, 900, 300}, kCost128 = {9000, 1425, 500}, kCost256 = {9500, 1600, 3000};

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

double cost_of(int side, int mode, int rows, int cols, int depth, int batch, int sms) {
    const Cost& c = side == 256 ? kCost256 : kCost128;
    return c.of(ceil_div(tile_count(mode, side, rows, cols) * batch, side == 256 ? sms / 2 : sms), depth);
}

template <int M>
int launch_gemm(const CUtensorMap& l, const CUtensorMap& r, const CUtensorMap& out, const Product& p, const Result& result,
                int batch, int sms, bool fine, cudaStream_t s) {
    const bool pair = !p.add && cost_of(256, M, p.rows, p.cols, p.depth, batch, sms) < cost_of(128, M, p.rows, p.cols, p.depth, batch, sms);
    if (fine)
        return pair ? launch_as<M, 256, true>(l, r, out, p, result, batch, sms, s)
                    : launch_as<M, 128, true>(l, r, out, p, result, batch, sms, s);
    return pair ? launch_as<M, 256, false>(l, r, out, p, result, batch, sms, s)
                : launch_as<M, 128, false>(l, r, out, p, result, batch, sms, s);
}

// What a step takes when all steps run in one kernel and when each product is a kernel;
// the cheaper way is taken.  Measured a call of five steps, one kernel against fifteen, 16-bit results (fp32): 72 against
// 114 us for one 192 x 192 matrix (80 against 129), 127 against 215 for 768 x 768 (137, 220), 119 against 136 for 40 of
// 192 x 192 (151, 151); 246 against 257 for 1024 x 1024 (278, 263), 168 against 163 for 12 of 384 x 384 (195, 168),
// 401 against 310 for 1100 x 1300 (458, 313).  Off by most at 900 x 900 bf16, where it takes 277 us for 239.
struct StepCost {
    int group;              // CTAs of a matrix in the one kernel
    double together, each;  // cycles of a step: one kernel, a kernel for each product
};
StepCost step_cost(int batch, int m, int n, bool squared, int sms) {
    const long long tiles = tile_count(kApply, 64, m, n), most = std::max(1LL, std::min<long long>(tiles, sms / batch));
    const long long group = ceil_div(tiles, ceil_div(tiles, most));  // no more than the rounds need
    const long long turns = ceil_div(batch, std::max(1LL, sms / group));
    const long long square = ceil_div(tile_count(kApply, 64, m, m), group);
    const double together = turns * (kCost64.of(square, n) + (squared ? kCost64.of(square, m) : 0) +
                                     kCost64.of(ceil_div(tiles, group), m));
    const auto apart = [&](int mode, int cols, int depth) {
        return std::min(cost_of(128, mode, m, cols, depth, batch, sms), cost_of(256, mode, m, cols, depth, batch, sms));
    };
    const double each = apart(kSymmetric, m, n) + (squared ? apart(kSymmetric, m, m) : 0) + apart(kApply, n, m);
    return {(int)group, together, each};
}

int type_bytes(int type) { return type == CIMEKV_F32 ? 4 : 2; }

// Whether every matrix begins on a multiple of `bytes`.
bool aligned(const Matrices& m, int batch, int bytes) {
    if (m.tabled) {
        for (int i = 0; i < batch; ++i)
            if ((uintptr_t)m.table[i] % bytes) return false;
        return true;
    }
    return (uintptr_t)m.base % bytes == 0 && (batch == 1 || m.batch_stride * type_bytes(m.type) % bytes == 0);
}

// Whether every row of every matrix can be read in vectors of four elements.
bool rows_in_fours(const Matrices& m, int batch, int cols) {
    if (!m.tabled && !m.base) return true;
    return cols % 4 == 0 && m.row_stride % 4 == 0 && aligned(m, batch, 4 * type_bytes(m.type));
}

// Everything after the arguments are checked: norms, X0, the steps, the result.
// share: the SMs to use, by all steps in one kernel; 0 for all SMs.
int run(PrepParams& prep, Result& result, int batch, int rows, int cols, int steps, float a, float b, float c,
        uint8_t* ws, int share, cudaStream_t s) {
    const Layout lay(batch, rows, cols);
    EncodeFn encode;
    int rc;
    int sms;
    if ((rc = encoder(&encode)) || (rc = sm_count(&sms))) return rc;
    if (share) sms = std::min(sms, share);
    __half* x[2] = {reinterpret_cast<__half*>(ws + lay.x0), reinterpret_cast<__half*>(ws + lay.x1)};
    __half* am = reinterpret_cast<__half*>(ws + lay.a);
    __half* pm = reinterpret_cast<__half*>(ws + lay.p);

    prep.rows = rows;
    prep.cols = cols;
    prep.transposed = rows > cols;
    prep.pitch = lay.xp;
    prep.plane = lay.x_plane;
    prep.parts = lay.parts;
    prep.part = reinterpret_cast<double*>(ws + lay.part);
    prep.arrivals = reinterpret_cast<unsigned*>(ws + lay.arrivals);
    prep.x = x[0];
    const bool vec = rows_in_fours(prep.g, batch, cols) && rows_in_fours(prep.mom, batch, cols);
    const bool flat = vec && (prep.g.row_stride == cols || rows == 1);
    if ((rc = cimekv_internal_no_pending_error()) || (rc = cimekv_internal_wait_word(CIMEKV_WAIT_PRODUCT, &result.lost)))
        return rc;
    const dim3 norm_grid(lay.parts, batch);
    if (flat) ns_norm_kernel<true><<<norm_grid, 256, 0, s>>>(prep);
    else ns_norm_kernel<false><<<norm_grid, 256, 0, s>>>(prep);
    if ((rc = launched("ns_norm_kernel"))) return rc;
    if (prep.transposed)
        rc = launch_chained("ns_prepare_tall_kernel", ns_prepare_tall_kernel,
                            dim3((cols + 63) / 64, (rows + 63) / 64, batch), 256, 0, 1, s, prep);
    else
        rc = launch_chained("ns_prepare_kernel", vec ? ns_prepare_kernel<true> : ns_prepare_kernel<false>,
                            dim3((cols + 255) / 256, (rows + 7) / 8, batch), 256, 0, 1, s, prep);
    if (rc) return rc;

    // sums of products of two planes are 2^24 times the value, planes 2^12 times
    const bool squared = c != 0.0f;
    const StepCost cost = step_cost(batch, lay.m, lay.n, squared, sms);
    const bool together = share || cost.together <= cost.each;  // all steps in one kernel
    // Fine sums where the result shows them: a 16-bit result's own rounding, 1e-3, hides the difference.  An fp32
    // parameter of 0.02 N after a step of 0.02 is off by 1.7e-7 with the coarse ones and by 0.9e-7 with the fine, as with
    // products in fp32 (48 of 768 x 768, where the products are kernels and the power limit hides the cost: 1,730 and 1,700
    // us).  In the one kernel of small matrices latency is all there is, and parameters take the coarse sums: 40 of 192 x 192
    // are off by 1.8e-7 in 125 us, by 1.2e-7 in 146 with fine sums (products in fp32 1.1e-7); with 10 of 192 x 768
    // beside them 180 and, with the polynomial as it stands too, 255 us.
    const bool fine = result.dst.type == CIMEKV_F32 && !(result.update && together);
    // Short sums are so exact that the completed square's rounding shows: on decaying spectra it leaves small matrices
    // further off than products in fp32 are, large ones (whose fp32 sums are long) not.  Off by, against fp32
    // products, completed and as it stands: 96 rows 1.33 and 0.87, 160 1.28 and 0.80, 192 1.13 and 0.70, 224 0.97
    // and 0.69, 256 1.00 and 0.67, 384 0.98 and 0.59, 768 0.74 and 0.49.  As it stands costs 192 x 192 74 us instead
    // of 68, 224 x 224 85 instead of 80, 48 of 768 x 768 a quarter: taken below the crossing.
    const bool plain = fine && squared && lay.m < 224;
    Steps st = {};
    Product &gram = st.product[0], &square = st.product[1], &apply = st.product[2];
    st.steps = steps;
    st.squared = squared;
    gram.rows = gram.cols = lay.m;
    gram.depth = lay.n;
    gram.alpha = (squared ? 1.0f : b) / kScale;
    gram.beta = (squared ? plain ? 0.0f : (float)(0.5 * b / c) : a) * kScale;
    if (squared) {
        square.rows = square.cols = square.depth = lay.m;
        square.alpha = c / kScale;
        square.beta = (plain ? a : (float)(a - 0.25 * (double)b * b / c)) * kScale;
    }
    if (plain) {
        square.add = am;
        square.add_plane = lay.a_plane;
        square.add_pitch = lay.ap;
        square.gamma = b / square.alpha;
    }
    apply.rows = apply.depth = lay.m;
    apply.cols = lay.n;
    apply.alpha = 1.0f / kScale;
    result.transposed = prep.transposed;
    result.vec = lay.n % 8 == 0 && aligned(result.dst, batch, 16);

    if (together) {
        const int group = cost.group;
        StepMaps maps;
        using T = Tile<64, true>;  // sizes are those of the fast one too
        constexpr int out_rows = T::kWarpRows;
        for (int i = 0; i < 2; ++i) {
            if ((rc = plane_map(encode, &maps.x[i], x[i], batch, lay.m, lay.n, lay.xp, 64))) return rc;
            if ((rc = plane_map(encode, &maps.x_out[i], x[i], batch, lay.m, lay.n, lay.xp, out_rows, true))) return rc;
        }
        if ((rc = plane_map(encode, &maps.b, am, batch, lay.m, lay.m, lay.ap, 64))) return rc;
        if ((rc = plane_map(encode, &maps.p, pm, batch, lay.m, lay.m, lay.ap, 64))) return rc;
        if ((rc = plane_map(encode, &maps.b_out, am, batch, lay.m, lay.m, lay.ap, out_rows, true))) return rc;
        if ((rc = plane_map(encode, &maps.p_out, pm, batch, lay.m, lay.m, lay.ap, out_rows, true))) return rc;
        static std::atomic<uint64_t> allowed[2];
        const auto kernel = fine ? ns_steps_kernel<true> : ns_steps_kernel<false>;
        if ((rc = allow_smem(kernel, T::smem(), allowed[fine]))) return rc;
        st.arrivals = prep.arrivals;
        st.group = group;
        const int most = sms / group;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(batch < most ? batch : most) * group);
        cfg.blockDim = dim3(T::kThreads);
        cfg.dynamicSmemBytes = T::smem();
        cfg.stream = s;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeCooperative;
        attr[0].val.cooperative = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, maps, st, result, batch);
        if (e == cudaSuccess) return CIMEKV_OK;
        (void)cudaGetLastError();
        return fail(CIMEKV_ECUDA, cudaGetErrorString(e));
    }
    // X as rows along K (Gram), as the right operand whose rows are K (apply), and to write
    CUtensorMap xleft[2], xright[2], xout[2], bmap, pmap, bout, pout;
    for (int i = 0; i < 2; ++i) {
        if ((rc = plane_map(encode, &xleft[i], x[i], batch, lay.m, lay.n, lay.xp, 128))) return rc;
        if ((rc = plane_map(encode, &xright[i], x[i], batch, lay.m, lay.n, lay.xp, kK))) return rc;
        if ((rc = plane_map(encode, &xout[i], x[i], batch, lay.m, lay.n, lay.xp, 32, true))) return rc;
    }
    if ((rc = plane_map(encode, &bmap, am, batch, lay.m, lay.m, lay.ap, 128))) return rc;
    if ((rc = plane_map(encode, &pmap, pm, batch, lay.m, lay.m, lay.ap, 128))) return rc;
    if ((rc = plane_map(encode, &bout, am, batch, lay.m, lay.m, lay.ap, 32, true))) return rc;
    if ((rc = plane_map(encode, &pout, pm, batch, lay.m, lay.m, lay.ap, 32, true))) return rc;
    for (int k = 0; k < steps; ++k) {
        if ((rc = launch_gemm<kSymmetric>(xleft[k & 1], xleft[k & 1], squared ? bout : pout, gram, result, batch, sms, fine, s))) return rc;
        if (squared && (rc = launch_gemm<kSymmetric>(bmap, bmap, pout, square, result, batch, sms, fine, s))) return rc;
        rc = k + 1 < steps ? launch_gemm<kApply>(pmap, xright[k & 1], xout[(k + 1) & 1], apply, result, batch, sms, fine, s)
                           : launch_gemm<kResult>(pmap, xright[k & 1], xout[0], apply, result, batch, sms, fine, s);
        if (rc) return rc;
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
    Result last = {};
    last.dst.base = out;
    last.dst.batch_stride = (long long)rows * cols;
    last.dst.type = type;
    return run(prep, last, batch, rows, cols, steps, a, b, c, static_cast<uint8_t*>(workspace), 0, (cudaStream_t)stream);
}

extern "C" int cimekv_muon_step(int count, void* const* params, const void* const* grads, float* const* momenta,
                                int p_type, int g_type, int rows, int cols, float lr, const float* lr_device,
                                float momentum, int nesterov, float weight_decay, float scale, int steps, float a,
                                float b, float c, float eps, void* workspace, size_t workspace_bytes, void* stream) {
    return cimekv_muon_step_on(0, count, params, grads, momenta, p_type, g_type, rows, cols, lr, lr_device, momentum,
                               nesterov, weight_decay, scale, steps, a, b, c, eps, workspace, workspace_bytes, stream);
}

// Which steps run side by side: those of small matrices, whose products are latency
// and leave SMs idle, and which run in one kernel (or nearly would; large ones fill the
// chip either way, and would hold their workspaces at the same time).  Every SM goes
// to the step that then takes longest.  Measured: 40 of 192 x 192 with 10 of 192 x 768 in
// 182 us a call, one after the other in 244.
extern "C" int cimekv_muon_shares(int groups, const int* counts, const int* rows, const int* cols, float c, int sms,
                                  int* shares) {
    int rc = cimekv_internal_begin_call();
    if (rc) return rc;
    if (groups < 0 || (groups && (!counts || !rows || !cols || !shares)))
        return fail(CIMEKV_EINVAL_SHAPE, "muon shares: null pointer or negative count");
    for (int i = 0; i < groups; ++i) {
        if (counts[i] < 0 || rows[i] < 0 || cols[i] < 0 || rows[i] > kMaxSide || cols[i] > kMaxSide)
            return fail(CIMEKV_EINVAL_SHAPE, "muon shares: bad size");
        shares[i] = 0;
    }
    if (sms < 0) return fail(CIMEKV_EINVAL_SHAPE, "muon shares: negative number of SMs");
    if (!sms && (rc = sm_count(&sms))) return rc;
    constexpr int kMost = 16;  // side by side
    int at[kMost], n = 0, left = sms;
    double alone[kMost], cost[kMost], all = 0.0;
    const auto of = [&](int i, int share) {
        const int batch = std::min(counts[i], kMaxTable);
        return step_cost(batch, std::min(rows[i], cols[i]), std::max(rows[i], cols[i]), c != 0.0f, share);
    };
    const auto calls = [&](int i) { return (double)ceil_div(counts[i], kMaxTable); };
    for (int i = 0; i < groups && n < kMost && sms >= 2 * kMost; ++i) {
        if (!counts[i] || !rows[i] || !cols[i]) continue;
        const StepCost one = of(i, sms);
        if (one.together > 1.25 * one.each) continue;
        all += alone[n] = calls(i) * std::min(one.together, one.each);
        at[n++] = i;
    }
    for (int k = 0; k < n; ++k) {  // half of the SMs by the times alone
        shares[at[k]] = std::max(2, (int)(0.5 * sms * alone[k] / all));
        left -= shares[at[k]];
        cost[k] = calls(at[k]) * of(at[k], shares[at[k]]).together;
    }
    double longest = 0.0;
    for (; n > 1; --left) {
        const int k = (int)(std::max_element(cost, cost + n) - cost);
        longest = cost[k];
        if (left <= 0) break;
        cost[k] = calls(at[k]) * of(at[k], ++shares[at[k]]).together;
    }
    // streams and events are about 10 us of the host's: a tenth has to be gained
    if (n < 2 || longest > 0.9 * all) std::fill(shares, shares + groups, 0);
    return CIMEKV_OK;
}

extern "C" int cimekv_muon_step_on(int share, int count, void* const* params, const void* const* grads,
                                   float* const* momenta, int p_type, int g_type, int rows, int cols, float lr,
                                   const float* lr_device, float momentum, int nesterov, float weight_decay, float scale,
                                   int steps, float a, float b, float c, float eps, void* workspace,
                                   size_t workspace_bytes, void* stream) {
    return cimekv_muon_step_weighted(share, count, params, grads, momenta, p_type, g_type, rows, cols, lr, lr_device,
                                     momentum, 1.0f - momentum, nesterov, weight_decay, scale, steps, a, b, c, eps, workspace,
                                     workspace_bytes, stream);
}

extern "C" int cimekv_muon_step_weighted(int share, int count, void* const* params, const void* const* grads,
                                         float* const* momenta, int p_type, int g_type, int rows, int cols, float lr,
                                         const float* lr_device, float momentum, float gain, int nesterov,
                                         float weight_decay, float scale, int steps, float a, float b, float c, float eps,
                                         void* workspace, size_t workspace_bytes, void* stream) {
    NvtxRange nvtx_range("cimekv_muon_step");
    int rc = cimekv_internal_begin_call();
    if (rc || (rc = check_iteration(count, rows, cols, steps, a, b, c, eps))) return rc;
    if (share < 0 || share == 1) return fail(CIMEKV_EINVAL_SHAPE, "muon step: a share is 0 (all) or at least 2 SMs");
    if (count > kMaxTable) return fail(CIMEKV_EINVAL_SHAPE, "muon step: too many matrices for one call");
    if (!valid_type(p_type) || !valid_type(g_type)) return fail(CIMEKV_EINVAL_SHAPE, "unknown element type");
    if (!(momentum >= 0.0f && momentum <= 1.0f)) return fail(CIMEKV_EINVAL_SHAPE, "momentum must be in [0, 1]");
    if (!std::isfinite(gain)) return fail(CIMEKV_EINVAL_SHAPE, "the gradient's weight must be finite");
    if (count == 0 || rows == 0 || cols == 0) return CIMEKV_OK;
    if (!params || !grads || !momenta) return fail(CIMEKV_EINVAL_SHAPE, "null pointer");
    for (int i = 0; i < count; ++i)
        if (!params[i] || !grads[i] || !momenta[i]) return fail(CIMEKV_EINVAL_SHAPE, "null pointer");
    // matrices written in one launch must not share memory (a gradient may be shared, but not with them)
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
    Result last = {};
    prep.g.tabled = prep.mom.tabled = last.dst.tabled = 1;
    prep.g.type = g_type;
    prep.mom.type = CIMEKV_F32;
    last.dst.type = p_type;
    prep.g.row_stride = prep.mom.row_stride = cols;
    for (int i = 0; i < count; ++i) {
        prep.g.table[i] = const_cast<void*>(grads[i]);
        prep.mom.table[i] = momenta[i];
        last.dst.table[i] = params[i];
    }
    prep.beta = momentum;
    prep.gain = gain;
    prep.nesterov = nesterov;
    prep.eps = eps;
    last.update = 1;
    last.lr = lr;
    last.lr_dev = lr_device;
    last.decay = weight_decay;
    last.scale = scale;
    return run(prep, last, count, rows, cols, steps, a, b, c, static_cast<uint8_t*>(workspace), share, (cudaStream_t)stream);
}
