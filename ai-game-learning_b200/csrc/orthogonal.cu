// Orthogonalising matrices by Newton-Schulz products, and the optimizer transition that uses it.
//
//   X0 = X / (|X|_F + eps),   X <- a X + (b G + c G^2) X with G = X X^T,   `steps` times,
//
// taken on the short side (a matrix with more rows than columns is transposed as it is read, and its
// result as it is written): X = U S V^T goes to U p(p(..p(S))) V^T with p(s) = a s + b s^3 + c s^5, whose
// iterates bring every singular value that is not tiny to about 1.  The transition (pbg_muon_step)
// orthogonalises each matrix's momentum and adds it to the matrix.
//
// A step is three products per matrix: A = X X^T, B = a I + b A + c A A (both symmetric: only the tiles
// on and above the diagonal are computed, the others mirrored, where there are more tiles than SMs), X' = B X,
// run on the tensor cores (tcgen05, fp32 accumulation in tensor memory) over all matrices of the call at once:
// one cooperative launch, a block per SM, or a pair of them on tiles of 256 x 256, with a grid barrier (1.3 us)
// between the 3 * steps products.  A matrix whose short side is at most 128 stays, with everything that is
// made of it, in the shared memory of a team of 1 to 8 blocks (orthogonalize_team_kernel).
//
// What bounds it.  4,096 x 4,096: the tensor cores, 1.29 PFLOP/s of fp16 products in three passes (3.30 ms; call
// after call the power cap makes it 3.9 ms).  14 of 256 x 1,024 (218 us): 15 products of a few microseconds each behind one
// another, so each one's first copies, last stores and the barrier.
//
// Precision.  16-bit operands alone are not enough: an error in X in the direction of a small singular
// value grows by a = 3.4 each step, so X is carried as a pair of fp16 numbers hi + lo of 2^14 X (22
// significant bits; every |x| <= sigma_max <= 2 keeps hi in range).  A and B are pairs too (2^13 A, 2^12 B)
// and each product takes three passes, hi hi + hi lo + lo hi, leaving errors of about 2^-22.  (Single fp16
// numbers for A and B where the output is bf16 took 1.85 ms at 4,096 x 4,096, but added up to as much error as
// the output's own rounding: 1.6e-3 of a noise matrix of 4,096 x 512.)  The tensor cores truncate as they
// accumulate, a bias that grows with the length of the sum (sums of 256 terms in three passes left 1.4e-5 of
// the result at 256 x 1024), so a sum is taken from tensor memory every 64 terms, the small products first,
// and added up in fp32 registers.
//
// Layout.  X, A and B live in the workspace as 128 x 64 tiles of 16 KB, hi then lo, already in the
// 128-byte-swizzled form that the tensor cores read from shared memory, so operands of any matrix of any
// size are fetched by plain contiguous bulk copies (no tensor maps), and one tile serves both as a
// K-major operand (X X^T) and, by halves, as an MN-major one (B X).  Short sides are padded with zeros to
// 128 and long sides to 64.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <math.h>
#include <string.h>

#include <algorithm>

#include "pbg_common.cuh"

namespace pbg {

constexpr int ORTHO_EPI_WARPS = 8;     // four row quarters x two column parts; 12 warps in all leave 168 registers
constexpr int ORTHO_PRODUCERS = 3;      // warps that issue bulk copies, a third of a stage's each
constexpr int ORTHO_THREADS = 32 * (1 + ORTHO_PRODUCERS + ORTHO_EPI_WARPS);  // warp 0 issues the products
constexpr int ORTHO_RING = 192 * 1024;  // operand stages
constexpr int ORTHO_STAGES = 8;         // at most
constexpr int ORTHO_BLOCK = 4096;       // an epilogue warp's staging block
constexpr int ORTHO_EYE = 2048;         // 16 rows of 128 bytes: (b / c) 2^13 I (2^13 I where c is 0) as three fp16 numbers, 32 bytes apart
constexpr int ORTHO_STAGING = ORTHO_EPI_WARPS * ORTHO_BLOCK;
constexpr int ORTHO_SMEM = 1024 + ORTHO_RING + ORTHO_STAGING + ORTHO_EYE;
constexpr int ORTHO_FLAT = 256;         // threads of the kernels around the products
constexpr int ORTHO_SPAN = ORTHO_FLAT * 16;  // elements whose squares one block sums
constexpr int ORTHO_TILE = 32768;       // bytes of a 128 x 64 tile, hi and lo
constexpr uint32_t ORTHO_WAIT_TRIES = 1u << 24;
// What the tensor cores take, on average, from sums whose large terms are positive (X X^T and A A), given back
// where the sums are scaled: each 16 terms truncate the running sum, so by 64 terms a Gram matrix comes out about
// 4 x 2^-24 of itself too small, by 16 or 32 terms 2 to 3 (measured on 1 to 1,536 rows of 7 to 4,096 columns).
// Five steps of 26 sizes and three spectra are then off by 0.02e-6 to 3.1e-6 of the result, 0.77 times what fp32
// products are on (geometric) average and 1.7 at most (33 x 2,000 of noise); with nothing given back by up to 3.6e-6.
constexpr float ORTHO_BACK_LONG = 1.0f + 0x1p-22f, ORTHO_BACK_SHORT = 1.0f + 0x1p-23f;
__device__ __forceinline__ float or_back(int terms) { return terms > 32 ? ORTHO_BACK_LONG : ORTHO_BACK_SHORT; }
constexpr float ORTHO_SX = 16384.0f, ORTHO_SA = 8192.0f, ORTHO_SB = 4096.0f;

struct OrthoDesc {
    int64_t src;     // first element
    int64_t ws;      // bytes of workspace before this matrix's tiles: X, X', A, B
    int64_t span0;   // spans, conversion tiles, symmetric and update tiles of the matrices before it
    int64_t conv0, sym0, upd0;
    int64_t gram0;   // its Gram matrix's items: tiles, each in `split` parts of its sum
    int64_t part0;   // items of the matrices before it whose sums are split
    int64_t slot0;   // blocks of the teams before it (short sides up to 128)
    int32_t m, n;    // short and long side
    int32_t team;    // blocks that work on it, where its short side is at most 128; else 0
    int32_t split;   // parts of the Gram matrix's sums
    int32_t tall;    // stored n x m
    float adjust;
};

struct OrthoArgs {
    const OrthoDesc* list;  // device, or null: `count` matrices like `one`, `one`'s sizes apart
    OrthoDesc one;
    int64_t one_src, one_ws, one_span, one_conv, one_sym, one_upd, one_gram;
    int64_t count, spans, convs, grams, syms, upds, slots;  // totals
    int bn_sym, bn_upd;  // output tile widths
    int pair;            // output tiles of 256 rows, by two blocks each
    int mirror;          // of A and B only what is on and above the diagonal is computed
    int steps;
    float a, b, c;
    double eps;
    // orthogonalize
    const void* x;
    int x_type;
    void* out;
    int out_type;
    // transition (x is null)
    float* grad;
    float* momentum;
    float* master;
    const float* controls;  // lr, momentum, decay, gradient scale
    int nesterov;
    uint32_t* bad;          // set where a direction is not finite: the transition leaves everything as it was
    // workspace
    double* sums;
    unsigned char* tiles;
    float* parts;           // of split sums: [item][row quarter][64 columns][column][lane]
    uint32_t* arrived;      // per item and epilogue warp, zero between uses
    uint32_t* barrier;
    uint32_t* error;
    int aligned;  // vector access to the flat buffers, x and out: 16 bytes at multiples of four elements
};

// ------------------------------------------------------------ tcgen05, mbarrier and bulk-copy access

__device__ __forceinline__ uint32_t or_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void or_mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void or_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void or_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool or_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
// bounded; also gives up when another role has
__device__ __forceinline__ bool or_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    for (uint32_t i = 0; i < ORTHO_WAIT_TRIES; ++i) {
        if (or_try_wait(bar, parity)) return true;
        if ((i & 1023u) == 1023u && *abort_flag) return false;
    }
    return false;
}
__device__ __forceinline__ void or_bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
// 128-byte-swizzled operand: K-major (rows of 128 bytes, 8-row atoms 1024 bytes apart), or MN-major (64
// columns of 8 k-rows an atom, the next k-rows 1024 bytes on, the next 64 columns `lbo` bytes on).  The low
// word of the descriptor, whose high word is the same for both.  (The address masked: in a cluster a block's
// shared addresses carry its rank above.)
__device__ __forceinline__ uint32_t or_desc(uint32_t addr, uint32_t lbo) { return ((addr >> 4) & 0x3FFFu) | ((lbo >> 4) << 16); }
// kind::f16: fp16 x fp16 -> fp32, M 128 or (pair) 256, A K-major, B K-major or MN-major
template <bool PAIR>
__device__ __forceinline__ uint32_t or_idesc(int n, int mn_major) {
    return (1u << 4) | ((uint32_t)mn_major << 16) | ((uint32_t)(n >> 3) << 17) | ((PAIR ? 16u : 8u) << 24);
}
template <bool PAIR>
__device__ __forceinline__ void or_mma(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    constexpr uint32_t high = (1024u >> 4) | (1u << 14) | (2u << 29);
    if constexpr (PAIR) {
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
            "mov.b64 da, {%1, %5};\n\t"
            "mov.b64 db, {%2, %5};\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
            "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(high)
            : "memory");
    } else {
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
            "mov.b64 da, {%1, %5};\n\t"
            "mov.b64 db, {%2, %5};\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
            "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(high)
            : "memory");
    }
}
// one lane of a converged warp; the compiler knows that it runs alone and keeps descriptors in uniform registers
__device__ __forceinline__ bool or_elect() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}
// the products issued so far arrive at a barrier when done; a pair's at both blocks' barriers
template <bool PAIR>
__device__ __forceinline__ void or_commit(uint32_t bar) {
    if constexpr (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                     "h"((uint16_t)3)
                     : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// Arrival at the pair's first block's barrier.  RELEASE: what the arriving thread has seen (its own block's copies
// landing in shared memory) is ordered before what the first block does after its wait.  Relaxed is for
// accumulators' columns that have been read: tcgen05.wait::ld and tcgen05.fence::before_thread_sync before the
// arrival, and fence::after_thread_sync after the wait, order tensor-memory accesses across a relaxed arrival.
template <bool RELEASE>
__device__ __forceinline__ void or_arrive_first(uint32_t bar) {
    if constexpr (RELEASE)
        asm volatile(
            "{\n\t.reg .b32 a;\n\t"
            "mapa.shared::cluster.u32 a, %0, 0;\n\t"
            "mbarrier.arrive.release.cluster.shared::cluster.b64 _, [a];\n\t}" ::"r"(bar)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .b32 a;\n\t"
            "mapa.shared::cluster.u32 a, %0, 0;\n\t"
            "mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [a];\n\t}" ::"r"(bar)
            : "memory");
}
// a wait for arrivals of the other block too
__device__ __forceinline__ bool or_try_wait_cluster(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
template <bool PAIR>
__device__ __forceinline__ bool or_wait_pair(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    for (uint32_t i = 0; i < ORTHO_WAIT_TRIES; ++i) {
        if (PAIR ? or_try_wait_cluster(bar, parity) : or_try_wait(bar, parity)) return true;
        if ((i & 1023u) == 1023u && *abort_flag) return false;
    }
    return false;
}
__device__ __forceinline__ void or_cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t or_cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void or_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void or_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void or_tmem_add16(uint32_t taddr, float* acc) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"  // with the load: the registers hold nothing before it
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[j] += __uint_as_float(r[j]);
}

// ------------------------------------------------------------ descriptors

__device__ __forceinline__ OrthoDesc or_get(const OrthoArgs& O, int64_t i) {
    if (O.list) return O.list[i];
    OrthoDesc d = O.one;
    d.src += i * O.one_src;
    d.ws += i * O.one_ws;
    d.span0 = i * O.one_span;
    d.conv0 = i * O.one_conv;
    d.sym0 = i * O.one_sym;
    d.upd0 = i * O.one_upd;
    d.gram0 = d.part0 = i * O.one_gram;
    d.slot0 = i * d.team;
    return d;
}

// the matrix that item t of the work counted by `field` belongs to (fields rise from 0)
__device__ __forceinline__ int64_t or_find(const OrthoArgs& O, int64_t t, int64_t OrthoDesc::*field, int64_t each) {
    if (!O.list) return t / each;
    int64_t lo = 0, hi = O.count - 1;
    while (lo < hi) {
        const int64_t mid = (lo + hi + 1) >> 1;
        if (O.list[mid].*field <= t) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__host__ __device__ __forceinline__ int or_mb(int m) { return (m + 127) >> 7; }
__host__ __device__ __forceinline__ int or_b64(int v) { return (v + 63) >> 6; }
// tiles from one row block to the next, odd: the blocks that read one column of tiles at a time would
// otherwise meet in a few memory slices where the pitch is a power of two (a row block of X has a tile to
// spare: a pair of blocks reads columns by 128)
__host__ __device__ __forceinline__ int or_pitch_x(int n) { return (or_b64(n) + 1) | 1; }
__host__ __device__ __forceinline__ int or_pitch_a(int m) { return 2 * or_mb(m) | 1; }
__host__ __device__ __forceinline__ int64_t or_x_bytes(int m, int n) { return (int64_t)or_mb(m) * or_pitch_x(n) * ORTHO_TILE; }
__host__ __device__ __forceinline__ int64_t or_a_bytes(int m) { return (int64_t)or_mb(m) * or_pitch_a(m) * ORTHO_TILE; }
// first column of the symmetric products' row block (pair of row blocks) i, and its tiles: from the diagonal on
// where the rest is mirrored
__host__ __device__ __forceinline__ int or_sym_first(int i, int pair, int mirror) { return mirror ? i * (pair ? 256 : 128) : 0; }
__host__ __device__ __forceinline__ int or_sym_row(int m, int i, int bn, int pair, int mirror) {
    return (or_b64(m) * 64 - or_sym_first(i, pair, mirror) + bn - 1) / bn;
}
__host__ __device__ __forceinline__ int or_row_blocks(int m, int pair) { return pair ? (or_mb(m) + 1) / 2 : or_mb(m); }

// ------------------------------------------------------------ the direction that is orthogonalised

__device__ __forceinline__ float or_load(const void* p, int type, int64_t i) {
    if (type == 0) return static_cast<const float*>(p)[i];
    if (type == 1) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    return __half2float(static_cast<const __half*>(p)[i]);
}

struct OrthoDirection {
    float mu, inv_scale;
    int nesterov;
};

__device__ __forceinline__ float or_momentum(const OrthoDirection& k, float g, float m) {
    return k.mu * m + (1.0f - k.mu) * (g * k.inv_scale);
}
__device__ __forceinline__ float or_direction(const OrthoDirection& k, float g, float m_new) {
    return k.nesterov ? k.mu * m_new + (1.0f - k.mu) * (g * k.inv_scale) : m_new;
}

__device__ __forceinline__ OrthoDirection or_controls(const OrthoArgs& O) {
    OrthoDirection k = {0.0f, 1.0f, O.nesterov};
    if (!O.x) {
        k.mu = O.controls[1];
        k.inv_scale = 1.0f / O.controls[3];
    }
    return k;
}

// the same sum in every thread, in an order that the block's size alone determines
__device__ __forceinline__ double or_block_sum(double v) {
    __shared__ double part[ORTHO_FLAT / 32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    double sum = 0.0;
#pragma unroll
    for (int w = 0; w < ORTHO_FLAT / 32; ++w) sum += part[w];
    return sum;
}

// what a matrix of that sum of squares is multiplied by: 2^14 over its norm and epsilon (a matrix of zeros stays
// zeros where epsilon is 0 too)
__device__ __forceinline__ double or_wide(const OrthoArgs& O, double squares) {
    const double norm = sqrt(squares) + O.eps;
    return norm == 0.0 ? 0.0 : (double)ORTHO_SX / norm;
}

// eight consecutive elements i .. i + 7, zeros from `live` on
__device__ __forceinline__ void or_load8(const void* p, int type, int64_t i, bool vector, int live, float* v) {
    if (vector && live >= 8) {
        if (type == 0) {
            const float4 f = __ldcg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + i));
            const float4 g = __ldcg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + i) + 1);
            v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w, v[4] = g.x, v[5] = g.y, v[6] = g.z, v[7] = g.w;
        } else {
            const uint2 f = __ldcg(reinterpret_cast<const uint2*>(static_cast<const unsigned short*>(p) + i));
            const uint2 g = __ldcg(reinterpret_cast<const uint2*>(static_cast<const unsigned short*>(p) + i) + 1);
            const uint32_t w[4] = {f.x, f.y, g.x, g.y};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 h = type == 1 ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[e]))
                                           : __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
                v[2 * e] = h.x, v[2 * e + 1] = h.y;
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < live ? or_load(p, type, i + e) : 0.0f;
    }
}

// Squares of each matrix's direction, a block and a sum per span (fp64: no overflow or underflow at any
// fp32 scale).
__global__ void __launch_bounds__(ORTHO_FLAT) orthogonalize_squares_kernel(const __grid_constant__ OrthoArgs O) {
    const OrthoDirection k = or_controls(O);
    const int64_t t = blockIdx.x;
    const OrthoDesc d = or_get(O, or_find(O, t, &OrthoDesc::span0, O.one_span));
    const int64_t total = (int64_t)d.m * d.n;
    const int64_t begin = (t - d.span0) * ORTHO_SPAN;
    const bool vector = O.aligned && d.src % 4 == 0;
    double sum = 0.0;
    bool bad = false;
    float g[2][8], m[2][8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int64_t i = begin + (h * ORTHO_FLAT + (int)threadIdx.x) * 8;
        const int live = i < total ? (int)(total - i < 8 ? total - i : 8) : 0;
        or_load8(O.x ? O.x : O.grad, O.x ? O.x_type : 0, d.src + i, vector, live, g[h]);
        if (!O.x) or_load8(O.momentum, 0, d.src + i, vector, live, m[h]);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float u = g[h][e];
            if (!O.x) {
                u = or_direction(k, u, or_momentum(k, u, m[h][e]));
                bad |= !isfinite(u);
            }
            sum += (double)u * (double)u;
        }
    if (bad) atomicExch(O.bad, 1u);
    sum = or_block_sum(sum);
    if (threadIdx.x == 0) O.sums[t] = sum;
}

__device__ __forceinline__ void or_split(float v, __half& hi, __half& lo) {
    hi = __float2half_rn(v);
    lo = __float2half_rn(v - __half2float(hi));
}

// The normalised direction as tiles of pairs, a block per tile (and the momentum, where there is one).  In
// the transition a direction that is not finite clears the matrices' gradients instead.
__global__ void __launch_bounds__(ORTHO_FLAT) orthogonalize_convert_kernel(const __grid_constant__ OrthoArgs O) {
    const OrthoDirection k = or_controls(O);
    const int64_t t = blockIdx.x;
    const OrthoDesc d = or_get(O, or_find(O, t, &OrthoDesc::conv0, O.one_conv));
    const int nb = or_b64(d.n);
    const int local = (int)(t - d.conv0);
    const int ti = local / nb, tj = local % nb;
    const bool clear = !O.x && *O.bad != 0u;
    double sum = 0.0;
    const int64_t spans = ((int64_t)d.m * d.n + ORTHO_SPAN - 1) / ORTHO_SPAN;
    for (int64_t i = threadIdx.x; i < spans; i += ORTHO_FLAT) sum += O.sums[d.span0 + i];
    const double wide = or_wide(O, or_block_sum(sum));
    const float scale = (float)wide;
    const bool plain = scale < 1.0e30f;  // beyond it belongs to a direction of (sub)normal smallness: in fp64 then
    unsigned char* tile = O.tiles + d.ws + ((int64_t)ti * or_pitch_x(d.n) + tj) * ORTHO_TILE;
    const bool vector = O.aligned && d.src % 4 == 0 && d.n % 4 == 0;
    // 1,024 chunks of 8 columns, four a thread.  Lanes run along rows of the stored matrix: 8 chunks of a row,
    // or (transposed) 32 rows of a chunk.
#pragma unroll 2
    for (int q = threadIdx.x; q < 1024; q += ORTHO_FLAT) {
        const int r = d.tall ? q & 127 : q >> 3, chunk = d.tall ? q >> 7 : q & 7;
        const int row = ti * 128 + r, col = tj * 64 + chunk * 8;
        const int live = row < d.m ? (d.n - col < 8 ? d.n - col : 8) : 0;
        const int64_t i = d.src + (d.tall ? (int64_t)col * d.m + row : (int64_t)row * d.n + col);
        const int64_t next = d.tall ? d.m : 1;
        if (clear) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < live) O.grad[i + e * next] = 0.0f;
            continue;
        }
        const void* src = O.x ? O.x : O.grad;
        const int type = O.x ? O.x_type : 0;
        float g[8], m[8];
        if (d.tall) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                g[e] = e < live ? or_load(src, type, i + e * next) : 0.0f;
                if (!O.x) m[e] = e < live ? O.momentum[i + e * next] : 0.0f;
            }
        } else {
            or_load8(src, type, i, vector, live, g);
            if (!O.x) or_load8(O.momentum, 0, i, vector, live, m);
        }
        if (!O.x) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                m[e] = or_momentum(k, g[e], m[e]);
                g[e] = or_direction(k, g[e], m[e]);
            }
            if (!d.tall && vector && live >= 8) {
                float4* p = reinterpret_cast<float4*>(O.momentum + i);
                p[0] = make_float4(m[0], m[1], m[2], m[3]);
                p[1] = make_float4(m[4], m[5], m[6], m[7]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e < live) O.momentum[i + e * next] = m[e];
            }
        }
        __align__(16) __half hi[8];
        __align__(16) __half lo[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) or_split(e < live ? (plain ? g[e] * scale : (float)((double)g[e] * wide)) : 0.0f, hi[e], lo[e]);
        const int at = r * 128 + ((chunk ^ (r & 7)) << 4);
        *reinterpret_cast<uint4*>(tile + at) = *reinterpret_cast<uint4*>(hi);
        *reinterpret_cast<uint4*>(tile + 16384 + at) = *reinterpret_cast<uint4*>(lo);
    }
}

// ------------------------------------------------------------ products

enum { OR_GRAM = 0, OR_SQUARE = 1, OR_UPDATE = 2 };

// one output tile: its matrix, row block, first column and width; the k-blocks of its sum that this item
// takes (`part` of `split`), and the first of its items among the split ones
struct OrthoTile {
    int which, i, c0, width, k0, kblocks, part, split;
    int64_t item;
};

// Tile (of the Gram matrix: item) t as one block (or the block of rank `rank` of a pair) sees it.  A pair's
// second row block may not exist (i = or_mb(m)); its columns come by 128.
template <bool PAIR, bool SPLIT>
__device__ __forceinline__ OrthoTile or_tile(const OrthoArgs& O, int kind, int64_t t, int rank) {
    OrthoTile T;
    const bool gram = SPLIT && kind == OR_GRAM;
    const int64_t w = gram                  ? or_find(O, t, &OrthoDesc::gram0, O.one_gram)
                      : kind != OR_UPDATE ? or_find(O, t, &OrthoDesc::sym0, O.one_sym)
                                          : or_find(O, t, &OrthoDesc::upd0, O.one_upd);
    T.which = (int)w;
    const OrthoDesc* d = O.list ? O.list + w : &O.one;
    const int64_t first = O.list ? (gram ? d->gram0 : kind != OR_UPDATE ? d->sym0 : d->upd0)
                                 : w * (gram ? O.one_gram : kind != OR_UPDATE ? O.one_sym : O.one_upd);
    const int m = d->m, n = d->n;
    int local = (int)(t - first);
    T.part = 0, T.split = 1, T.k0 = 0, T.item = 0;
    if (gram && d->split > 1) {
        T.split = d->split;
        T.part = local % T.split;
        local /= T.split;
        T.item = (O.list ? d->part0 : first) + (int64_t)local * T.split;
    }
    if (kind != OR_UPDATE) {
        T.i = 0;
        for (int r; local >= (r = or_sym_row(m, T.i, O.bn_sym, PAIR, O.mirror)); ++T.i) local -= r;
        T.c0 = or_sym_first(T.i, PAIR, O.mirror) + local * O.bn_sym;
        T.width = min(O.bn_sym, or_b64(m) * 64 - T.c0);
    } else {
        const int across = (or_b64(n) * 64 + O.bn_upd - 1) / O.bn_upd;
        T.i = local / across;
        T.c0 = (local % across) * O.bn_upd;
        T.width = min(O.bn_upd, or_b64(n) * 64 - T.c0);
    }
    if (PAIR) {
        T.i = 2 * T.i + rank;
        T.width = (T.width + 127) & ~127;
    }
    if (kind == OR_SQUARE && O.c == 0.0f) {
        T.kblocks = T.width >> 6;  // no square: only the tile's own columns of A
    } else {
        T.kblocks = or_b64(kind == OR_GRAM ? n : m);
        if (T.split > 1) {
            T.k0 = (int)((int64_t)T.kblocks * T.part / T.split);
            T.kblocks = (int)((int64_t)T.kblocks * (T.part + 1) / T.split) - T.k0;
        }
    }
    return T;
}

// where a matrix's tiles lie at a step
struct OrthoPlace {
    int64_t x_row, a_row;  // bytes of a row block
    unsigned char *x, *x_next, *a, *b;
};
__device__ __forceinline__ OrthoPlace or_place(const OrthoArgs& O, const OrthoDesc& d, int step) {
    OrthoPlace L;
    const int64_t xb = or_x_bytes(d.m, d.n);
    L.x_row = (int64_t)or_pitch_x(d.n) * ORTHO_TILE;
    L.a_row = (int64_t)or_pitch_a(d.m) * ORTHO_TILE;
    unsigned char* base = O.tiles + d.ws;
    L.x = base + (step & 1 ? xb : 0);
    L.x_next = base + (step & 1 ? 0 : xb);
    L.a = base + 2 * xb;
    L.b = L.a + or_a_bytes(d.m);
    return L;
}

// A thread's 64 finished values of one row as a row of a 128 x 64 tile, hi then lo, by way of the warp's
// staging block of 32 rows (rows of 128 bytes are contiguous in the tile, so each part is one bulk copy); lo
// has a block of its own where the warp of the other column part has no columns (`spare`).
__device__ __forceinline__ void or_store_rows(uint32_t blk, uint32_t spare, unsigned char* dst, int lane, float* v) {
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();
#pragma unroll 1
    for (int low = 0; low < 2; ++low) {
        const uint32_t at = low && spare ? spare : blk;
        if (low && !spare) {
            if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            __syncwarp();
        }
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                // opaque, or the conversions of both parts would be made and kept before the first
                asm volatile("" : "+f"(v[8 * q + 2 * j]), "+f"(v[8 * q + 2 * j + 1]));
                const float x0 = v[8 * q + 2 * j], x1 = v[8 * q + 2 * j + 1];
                __half2 h = __floats2half2_rn(x0, x1);
                if (low) {
                    const float2 f = __half22float2(h);
                    h = __floats2half2_rn(x0 - f.x, x1 - f.y);
                }
                w[j] = *reinterpret_cast<uint32_t*>(&h);
            }
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + (uint32_t)lane * 128u + (uint32_t)((q ^ (lane & 7)) << 4)),
                         "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                         : "memory");
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
            asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst + (low ? 16384 : 0)), "r"(at), "r"(4096u)
                         : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
    }
}

// one finished value at element i of the output, or into the master
struct OrthoOut {
    float lr, shrink;  // of the transition
};
__device__ __forceinline__ void or_write_one(const OrthoArgs& O, const OrthoOut& k, int64_t i, float v) {
    if (!O.x) O.master[i] = O.master[i] * k.shrink - k.lr * v;
    else if (O.out_type == 0) static_cast<float*>(O.out)[i] = v;
    else if (O.out_type == 1) static_cast<__nv_bfloat16*>(O.out)[i] = __float2bfloat16_rn(v);
    else static_cast<__half*>(O.out)[i] = __float2half_rn(v);
}

// The last update: 64 columns of a warp's 32 rows to the output or the master, 32 columns at a time by way
// of the warp's staging block (32 rows of 128 bytes, chunks swizzled by the row), so that lanes are
// neighbours in memory whichever side is stored along.  Loops are kept rolled: each launch runs this once, and
// unrolled its instructions took longer to fetch (12 us) than to run.  v is used up.
__device__ __forceinline__ void or_finish_out(const OrthoArgs& O, int which, int row, int cb, uint32_t blk, int lane, float* v) {
    const OrthoDesc d = or_get(O, which);
    const int r0 = row - lane;
    OrthoOut k = {0.0f, 1.0f};
    if (!O.x) {
        k.lr = O.controls[0];
        k.shrink = 1.0f - k.lr * O.controls[2];
        k.lr *= d.adjust;
    }
    const float scale = 1.0f / (ORTHO_SB * ORTHO_SX);
    const bool vector = d.n % 4 == 0 && d.src % 4 == 0 && O.aligned;
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int q = 0; q < 8; ++q)
            asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(blk + (uint32_t)lane * 128u + (uint32_t)((q ^ (lane & 7)) << 4)),
                         "f"(v[4 * q] * scale), "f"(v[4 * q + 1] * scale), "f"(v[4 * q + 2] * scale), "f"(v[4 * q + 3] * scale)
                         : "memory");
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = v[j + 32];
        __syncwarp();
        const int col0 = cb * 64 + half * 32;
        if (d.tall) {  // a column of the tile is a run in memory: a lane per row
            const int cols = min(32, d.n - col0);
            if (row < d.m) {
#pragma unroll 1
                for (int j0 = 0; j0 < cols; j0 += 4) {
                    const int64_t at = d.src + (int64_t)(col0 + j0) * d.m + row;
                    float x[4], w[4];
                    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                                 : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3])
                                 : "r"(blk + (uint32_t)lane * 128u + (uint32_t)(((j0 >> 2) ^ (lane & 7)) << 4))
                                 : "memory");
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (!O.x && j0 + j < cols) w[j] = O.master[at + (int64_t)j * d.m];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (j0 + j >= cols) continue;
                        if (!O.x) O.master[at + (int64_t)j * d.m] = w[j] * k.shrink - k.lr * x[j];
                        else or_write_one(O, k, at + (int64_t)j * d.m, x[j]);
                    }
                }
            }
        } else {  // eight lanes a row, four columns each
            const int col = col0 + (lane & 7) * 4;
            const int rows = min(32, d.m - r0);
#pragma unroll 1
            for (int r1 = lane >> 3; r1 < rows; r1 += 8) {
                float x[2][4];
                float4 w[2];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int r = r1 + 4 * u;
                    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                                 : "=f"(x[u][0]), "=f"(x[u][1]), "=f"(x[u][2]), "=f"(x[u][3])
                                 : "r"(blk + (uint32_t)r * 128u + (uint32_t)(((lane & 7) ^ (r & 7)) << 4))
                                 : "memory");
                    if (!O.x && vector && r < rows && col < d.n)
                        w[u] = *reinterpret_cast<const float4*>(O.master + d.src + (int64_t)(r0 + r) * d.n + col);
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int r = r1 + 4 * u;
                    const int64_t at = d.src + (int64_t)(r0 + r) * d.n + col;
                    if (r >= rows || col >= d.n) continue;
                    if (!vector) {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (col + j < d.n) or_write_one(O, k, at + j, x[u][j]);
                    } else if (!O.x) {
                        *reinterpret_cast<float4*>(O.master + at) =
                            make_float4(w[u].x * k.shrink - k.lr * x[u][0], w[u].y * k.shrink - k.lr * x[u][1],
                                        w[u].z * k.shrink - k.lr * x[u][2], w[u].w * k.shrink - k.lr * x[u][3]);
                    } else if (O.out_type == 0) {
                        *reinterpret_cast<float4*>(static_cast<float*>(O.out) + at) = make_float4(x[u][0], x[u][1], x[u][2], x[u][3]);
                    } else {
                        uint2 b;
                        if (O.out_type == 1) {
                            const __nv_bfloat162 p = __floats2bfloat162_rn(x[u][0], x[u][1]), q = __floats2bfloat162_rn(x[u][2], x[u][3]);
                            b.x = *reinterpret_cast<const uint32_t*>(&p), b.y = *reinterpret_cast<const uint32_t*>(&q);
                        } else {
                            const __half2 p = __floats2half2_rn(x[u][0], x[u][1]), q = __floats2half2_rn(x[u][2], x[u][3]);
                            b.x = *reinterpret_cast<const uint32_t*>(&p), b.y = *reinterpret_cast<const uint32_t*>(&q);
                        }
                        *reinterpret_cast<uint2*>(static_cast<unsigned short*>(O.out) + at) = b;
                    }
                }
            }
        }
        __syncwarp();
    }
}

// A launch of the products has one scaled identity: a list's few matrices of at most 32 rows take the others'.
__device__ __forceinline__ float or_square_back(const OrthoArgs& O) { return O.list ? ORTHO_BACK_LONG : or_back(O.one.m); }
// What the square's sum A A + A (b / factor) I is multiplied by; where there is no square, b.
__device__ __forceinline__ float or_square_factor(const OrthoArgs& O, float back) { return O.c != 0.0f ? O.c * back : O.b; }

// what an epilogue warp does with its 32 rows x 64 columns (rows row - lane ..., column block cb of 64)
__device__ __forceinline__ void or_finish(const OrthoArgs& O, int kind, int step, int which, int i, int row, int cb,
                                          uint32_t blk, uint32_t spare, int lane, float* v) {
    const OrthoPlace L = or_place(O, or_get(O, which), step);
    const int r0 = row - lane;
    if (kind == OR_UPDATE) {
#pragma unroll
        for (int j = 0; j < 64; ++j) v[j] *= 1.0f / ORTHO_SB;
        unsigned char* tile = L.x_next + i * L.x_row + (int64_t)cb * ORTHO_TILE + (r0 & 127) * 128;
        or_store_rows(blk, spare, tile, lane, v);
        return;
    }
    if (O.mirror && (cb >> 1) < i) return;  // below the diagonal (a pair's second row block): mirrored from above
    unsigned char* dst = kind == OR_GRAM ? L.a : L.b;
    const float factor = kind == OR_GRAM ? ORTHO_BACK_LONG * (ORTHO_SA / (ORTHO_SX * ORTHO_SX))
                                         : or_square_factor(O, or_square_back(O)) * (ORTHO_SB / (ORTHO_SA * ORTHO_SA));
    const float diagonal = kind == OR_GRAM ? 0.0f : O.a * ORTHO_SB;
#pragma unroll
    for (int j = 0; j < 64; ++j) v[j] = fmaf(v[j], factor, row == cb * 64 + j ? diagonal : 0.0f);
    unsigned char* tile = dst + i * L.a_row + (int64_t)cb * ORTHO_TILE + (r0 & 127) * 128;
    or_store_rows(blk, spare, tile, lane, v);
    if (O.mirror && cb * 64 >= (i + 1) * 128) {
        // the mirrored place of (row, cb * 64 + j): row block cb / 2, column block row / 64, row (cb & 1) * 64 + j
        // of that tile; lanes are neighbours
        const int mc = row & 63;
        unsigned char* mt = dst + (int64_t)(cb >> 1) * L.a_row + (int64_t)(row >> 6) * ORTHO_TILE + (cb & 1) * 8192 + (mc & 7) * 2;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            unsigned char* at = mt + j * 128 + (((mc >> 3) ^ j) << 4);
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                __half hi, lo;
                or_split(v[8 * q + j], hi, lo);
                *reinterpret_cast<__half*>(at + q * 1024) = hi;
                *reinterpret_cast<__half*>(at + q * 1024 + 16384) = lo;
            }
        }
    }
}

// The scaled identity that b A is taken against, from its row `first` on, by 128 threads: 16 rows x 8 chunks of
// 16 bytes, swizzled; chunks 0-1 hold the value's first part (columns 0-15), 2-3 and 4-5 what the parts before
// leave.  Three parts hold the value to 33 bits.  (Two left b off by 1.0e-7 of itself, the same way in every
// step: matrices of 3 x 500 came out 2.1e-6 off, where fp32 products are 7e-7.)
__device__ __forceinline__ void or_identity(const OrthoArgs& O, unsigned char* eye, int t, int first, float back) {
    const int r = t >> 3, chunk = t & 7;
    const double value = O.c != 0.0f ? (double)O.b / (double)or_square_factor(O, back) * ORTHO_SA : ORTHO_SA;
    __half part[3];
    double left = value;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        part[i] = __double2half(left);
        left -= (double)__half2float(part[i]);
    }
    const __half zero = __float2half_rn(0.0f), mine = chunk < 2 ? part[0] : chunk < 4 ? part[1] : chunk < 6 ? part[2] : zero;
    __align__(16) __half h[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = (chunk & 1) * 8 + e == r + first ? mine : zero;
    *reinterpret_cast<uint4*>(eye + r * 128 + ((chunk ^ (r & 7)) << 4)) = *reinterpret_cast<uint4*>(h);
}

// c A A + b A = c (A A + A (b / c) I): 16 columns of A (hi and lo) against the scaled identity, added at d; the
// products that are small beside the sum go before its large ones, whose size decides what truncation takes
template <bool PAIR>
__device__ __forceinline__ void or_identity_small(uint32_t d, uint32_t a, uint32_t al, uint32_t eye, uint32_t idesc) {
    or_mma<PAIR>(d, a, eye + 4, idesc, 1u);
    or_mma<PAIR>(d, al, eye + 2, idesc, 1u);
    or_mma<PAIR>(d, a, eye + 2, idesc, 1u);
    or_mma<PAIR>(d, al, eye, idesc, 1u);
}

struct OrthoShared {
    uint64_t full[ORTHO_STAGES], empty[ORTHO_STAGES], peer[ORTHO_STAGES], acc_full[4], acc_empty[4], done;
    uint32_t tmem;
    int ok;
    volatile int abort_flag;
};

// Between two phases: every role of every block arrives (the launch is cooperative, so all blocks run);
// bounded.  False when the wait, or a role of any block, gave up (the word's top bit).
__device__ __forceinline__ bool or_phase_end(const OrthoArgs& O, OrthoShared& S, uint32_t phases) {
    asm volatile("fence.proxy.async;" ::: "memory");
    asm volatile("bar.sync 1, %0;" ::"n"(ORTHO_THREADS) : "memory");
    if (threadIdx.x == 0) {
        const uint32_t target = phases * gridDim.x;
        if (S.abort_flag) atomicOr(O.barrier, 0x80000000u);
        asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(O.barrier) : "memory");
        uint32_t seen = 0;
        for (uint32_t i = 0; seen < target && i < ORTHO_WAIT_TRIES; ++i)
            asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(O.barrier) : "memory");
        if (seen < target) atomicCAS(O.error, 0u, 4u);
        S.ok = seen >= target && !(seen & 0x80000000u);
    }
    asm volatile("bar.sync 1, %0;" ::"n"(ORTHO_THREADS) : "memory");
    asm volatile("fence.proxy.async;" ::: "memory");
    return *reinterpret_cast<volatile int*>(&S.ok) != 0;
}

// The operand stages of a kind of product: the row operand's tile, hi and lo, then up to four (of a pair, two:
// half of the columns) 64-wide pieces of the other operand, hi parts and lo parts.
struct OrthoStage {
    int stages;
    uint32_t b_part, bytes;
};
template <bool PAIR>
__device__ __forceinline__ OrthoStage or_stage(int bn) {
    OrthoStage G;
    G.b_part = (uint32_t)(PAIR ? bn / 2 : bn) * 128u;
    G.bytes = ORTHO_TILE + 2 * G.b_part;
    G.stages = min(ORTHO_STAGES, (int)(ORTHO_RING / G.bytes));
    return G;
}

// Accumulators in tensor memory, as a power of two: four where no tile is wider than 128 (a short k-block's
// products take less time than an accumulator's way to the registers), else two.
__device__ __forceinline__ uint32_t or_buffers(const OrthoArgs& O) { return max(O.bn_sym, O.bn_upd) <= 128 ? 2u : 1u; }

// A producer warp's elected lane, one phase.  A stage is copy 0, the row operand, and copies 1 .. 8 at most, a
// 64-row or 64-column piece of the other operand each, hi or lo; the producer warps take them in turn.  `pipe`:
// parity of each stage's next use, a bit a stage, kept from phase to phase.
template <bool PAIR, bool SPLIT>
__device__ __forceinline__ void or_produce(const OrthoArgs& O, OrthoShared& S, uint32_t ring, int kind, int step, int rank,
                                           int producer, uint32_t& pipe) {
    const int64_t tiles = SPLIT && kind == OR_GRAM ? O.grams : kind != OR_UPDATE ? O.syms : O.upds;
    const OrthoStage G = or_stage<PAIR>(kind == OR_UPDATE ? O.bn_upd : O.bn_sym);
    const uint32_t full0 = or_smem(&S.full[0]), empty0 = or_smem(&S.empty[0]);
    bool ok = true;
    int s = 0;
    uint32_t used = 0;
    for (int64_t t = PAIR ? blockIdx.x >> 1 : blockIdx.x; ok && t < tiles; t += PAIR ? gridDim.x >> 1 : gridDim.x) {
        OrthoTile T = or_tile<PAIR, SPLIT>(O, kind, t, rank);
        const int kblocks = T.kblocks, pieces = T.width >> (PAIR ? 7 : 6);
        const OrthoDesc desc = or_get(O, T.which);
        const OrthoPlace L = or_place(O, desc, step);
        if (PAIR) T.i = min(T.i, or_mb(desc.m) - 1);  // the row block that is not there: any other, never stored
        const unsigned char* src[3];  // of k-blocks 0 and 1
        uint32_t dst[3], bytes[3], expect = 0;
        // what an odd k-block and a pair of them add to the pieces (to copy 0: one tile each)
        const int64_t odd = kind == OR_UPDATE ? 8192 : ORTHO_TILE, pair = kind == OR_UPDATE ? L.x_row : 2 * ORTHO_TILE;
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            const int copy = q * ORTHO_PRODUCERS + producer;
            if (copy == 0) {
                src[q] = kind == OR_GRAM ? L.x + T.i * L.x_row : kind == OR_SQUARE ? L.a + T.i * L.a_row : L.b + T.i * L.a_row;
                if (kind == OR_SQUARE && O.c == 0.0f) src[q] += (int64_t)(T.c0 >> 6) * ORTHO_TILE;
                dst[q] = 0, bytes[q] = ORTHO_TILE;
            } else {
                const int piece = (copy - 1) >> 1, part = (copy - 1) & 1;
                const int cb = (T.c0 >> 6) + (PAIR ? rank * pieces : 0) + piece;
                dst[q] = ORTHO_TILE + part * G.b_part + piece * 8192u;
                bytes[q] = piece < pieces ? 8192u : 0u;
                if (kind == OR_UPDATE) src[q] = L.x + (int64_t)cb * ORTHO_TILE + part * 16384;  // 64 k-rows of column block cb
                else src[q] = (kind == OR_GRAM ? L.x + (cb >> 1) * L.x_row : L.a + (cb >> 1) * L.a_row) + (cb & 1) * 8192 + part * 16384;
            }
            if (SPLIT) src[q] += (int64_t)T.k0 * ORTHO_TILE;
            expect += bytes[q];
        }
        for (int kb = 0; kb < kblocks; ++kb) {
            if (!or_wait(empty0 + 8 * s, ((pipe >> s) & 1u) ^ 1u, &S.abort_flag)) {
                ok = false;
                break;
            }
            pipe ^= 1u << s;
            used |= 1u << s;
            const uint32_t bar = full0 + 8 * s, at = ring + s * G.bytes;
            or_expect_tx(bar, expect);
#pragma unroll
            for (int q = 0; q < 3; ++q) {
                const bool row = q == 0 && producer == 0;
                if (bytes[q]) or_bulk_load(at + dst[q], src[q] + (kb & 1 ? (row ? ORTHO_TILE : odd) : 0), bytes[q], bar);
                if (kb & 1) src[q] += row ? 2 * ORTHO_TILE : pair;
            }
            if (++s == G.stages) s = 0;
        }
    }
    if (!ok) {
        atomicCAS(O.error, 0u, 1u);
        S.abort_flag = 1;
    }
    if (S.abort_flag) {  // every copy under way lands before the block can end
        for (int q = 0; q < G.stages; ++q)
            for (uint32_t i = 0; ((used >> q) & 1u) && i < ORTHO_WAIT_TRIES &&
                                 !or_try_wait(full0 + 8 * q, ((pipe >> q) & 1u) ^ 1u); ++i) {
            }
    }
}

// The issuing warp's elected lane (of a pair's first block), one phase.  `acc` counts accumulators used.
template <bool PAIR, bool SPLIT>
__device__ __forceinline__ void or_issue(const OrthoArgs& O, OrthoShared& S, uint32_t ring, int kind, uint32_t& pipe,
                                         uint32_t& acc) {
    const int64_t tiles = SPLIT && kind == OR_GRAM ? O.grams : kind != OR_UPDATE ? O.syms : O.upds;
    const OrthoStage G = or_stage<PAIR>(kind == OR_UPDATE ? O.bn_upd : O.bn_sym);
    const uint32_t full0 = or_smem(&S.full[0]), empty0 = or_smem(&S.empty[0]);
    const uint32_t peer0 = or_smem(&S.peer[0]);
    const uint32_t acc_full0 = or_smem(&S.acc_full[0]), acc_empty0 = or_smem(&S.acc_empty[0]);
    const bool linear = kind == OR_SQUARE && O.c == 0.0f;
    const int chunk = linear ? 1 << 20 : 1;
    const int mn = kind == OR_UPDATE;
    const uint32_t b_step = mn ? 2048u >> 4 : 32u >> 4, lbo = mn ? 8192u : 16u;
    const uint32_t eye = or_desc(ring + ORTHO_RING + ORTHO_STAGING, 16), eye_idesc = or_idesc<PAIR>(16, 0);
    const uint32_t tmem = S.tmem, shift = or_buffers(O), buffers = 1u << shift;
    bool ok = true;
    int s = 0;
    for (int64_t t = PAIR ? blockIdx.x >> 1 : blockIdx.x; ok && t < tiles; t += PAIR ? gridDim.x >> 1 : gridDim.x) {
        const OrthoTile T = or_tile<PAIR, SPLIT>(O, kind, t, 0);
        const int kblocks = T.kblocks;
        const uint32_t idesc = or_idesc<PAIR>(T.width, mn);
        const int eye0 = kind == OR_SQUARE ? T.c0 >> 6 : 1 << 30, eye1 = eye0 + (T.width >> 6);
        for (int k0 = 0; ok && k0 < kblocks; k0 += chunk, ++acc) {
            const uint32_t b = acc & (buffers - 1u);
            if (!or_wait_pair<PAIR>(acc_empty0 + 8 * b, ((acc >> shift) & 1u) ^ 1u, &S.abort_flag)) {
                ok = false;
                break;
            }
            or_fence_after();
            const uint32_t d = tmem + b * (512u >> shift);
            const int k1 = min(k0 + chunk, kblocks);
            for (int kb = k0; kb < k1; ++kb) {
                if (!or_wait(full0 + 8 * s, (pipe >> s) & 1u, &S.abort_flag) ||
                    (PAIR && !or_wait_pair<PAIR>(peer0 + 8 * s, (pipe >> s) & 1u, &S.abort_flag))) {
                    ok = false;
                    break;
                }
                pipe ^= 1u << s;
                or_fence_after();
                const uint32_t a = or_desc(ring + s * G.bytes, 16), al = a + (16384u >> 4);
                const uint32_t bh = or_desc(ring + s * G.bytes + ORTHO_TILE, lbo), bl = bh + (G.b_part >> 4);
                if (linear) {
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) {
                        const uint32_t dd = d + (uint32_t)kb * 64u + ks * 16;
                        or_mma<PAIR>(dd, al + ks * 2, eye, eye_idesc, 0u);
                        or_mma<PAIR>(dd, a + ks * 2, eye, eye_idesc, 1u);
                    }
                } else {
                    // the small products first: they are added to a small sum
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) or_mma<PAIR>(d, al + ks * 2, bh + ks * b_step, idesc, ks > 0);
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) or_mma<PAIR>(d, a + ks * 2, bl + ks * b_step, idesc, 1u);
                    const bool diagonal = kb >= eye0 && kb < eye1;  // this k-block's columns once more, 16 at a time
                    const uint32_t dd = d + (uint32_t)(kb - eye0) * 64u;
                    if (diagonal) {
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks) or_identity_small<PAIR>(dd + ks * 16, a + ks * 2, al + ks * 2, eye, eye_idesc);
                    }
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) or_mma<PAIR>(d, a + ks * 2, bh + ks * b_step, idesc, 1u);
                    if (diagonal) {
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks) or_mma<PAIR>(dd + ks * 16, a + ks * 2, eye, eye_idesc, 1u);
                    }
                }
                or_commit<PAIR>(empty0 + 8 * s);
                if (++s == G.stages) s = 0;
            }
            if (ok) or_commit<PAIR>(acc_full0 + 8 * b);
        }
    }
    if (!ok) {
        atomicCAS(O.error, 0u, 2u);
        S.abort_flag = 1;
    }
}

// The same warp of a pair's second block: tells the first when a stage's copies have landed here.
__device__ __forceinline__ void or_relay(const OrthoArgs& O, OrthoShared& S, int kind, uint32_t& pipe) {
    constexpr bool PAIR = true, SPLIT = false;
    const int64_t tiles = SPLIT && kind == OR_GRAM ? O.grams : kind != OR_UPDATE ? O.syms : O.upds;
    const OrthoStage G = or_stage<PAIR>(kind == OR_UPDATE ? O.bn_upd : O.bn_sym);
    const uint32_t full0 = or_smem(&S.full[0]), peer0 = or_smem(&S.peer[0]);
    bool ok = true;
    int s = 0;
    for (int64_t t = PAIR ? blockIdx.x >> 1 : blockIdx.x; ok && t < tiles; t += PAIR ? gridDim.x >> 1 : gridDim.x) {
        const int kblocks = or_tile<PAIR, SPLIT>(O, kind, t, 1).kblocks;
        for (int kb = 0; kb < kblocks; ++kb) {
            if (!or_wait(full0 + 8 * s, (pipe >> s) & 1u, &S.abort_flag)) {
                ok = false;
                break;
            }
            pipe ^= 1u << s;
            or_arrive_first<true>(peer0 + 8 * s);
            if (++s == G.stages) s = 0;
        }
    }
    if (!ok) {
        atomicCAS(O.error, 0u, 6u);
        S.abort_flag = 1;
    }
}

// A part of a split sum (an epilogue warp's rows and columns): to the workspace, and, where it is the last of
// its tile's parts to arrive, the sum of all parts in order, so that the result does not depend on who is last.
__device__ __forceinline__ bool or_join(const OrthoArgs& O, const OrthoTile& T, int e, int quad, int group0, int groups, int lane,
                                        float* v) {
    const int64_t next = (int64_t)128 * O.bn_sym;  // between a tile's parts
    float* first = O.parts + T.item * next + ((int64_t)quad * (O.bn_sym >> 6) + group0) * 2048 + lane;
    float* mine = first + T.part * next;
#pragma unroll
    for (int j = 0; j < 128; ++j)
        if (j < 64 * groups) __stcg(mine + j * 32, v[j]);
    __threadfence();
    __syncwarp();
    uint32_t* arrived = O.arrived + T.item * ORTHO_EPI_WARPS + e;
    uint32_t before = 0;
    if (lane == 0) before = atomicAdd(arrived, 1u);
    if (__shfl_sync(0xffffffffu, before, 0) != (uint32_t)T.split - 1u) return false;
    __threadfence();
    if (lane == 0) *arrived = 0u;
#pragma unroll
    for (int j = 0; j < 128; ++j)
        if (j < 64 * groups) v[j] = __ldcg(first + j * 32);
    for (int p = 1; p < T.split; ++p) {
        const float* part = first + p * next;
#pragma unroll
        for (int j = 0; j < 128; ++j)
            if (j < 64 * groups) v[j] += __ldcg(part + j * 32);
    }
    return true;
}

// An epilogue warp, one phase: a quarter of the rows, one or (tiles wider than 128) two groups of 64
// columns of each tile.
template <bool PAIR, bool SPLIT>
__device__ __forceinline__ void or_collect(const OrthoArgs& O, OrthoShared& S, uint32_t ring, int kind, int step, int rank, int e,
                                           uint32_t& acc) {
    const int lane = threadIdx.x & 31, quad = (threadIdx.x >> 5) & 3, part = e >> 2;
    const int64_t tiles = SPLIT && kind == OR_GRAM ? O.grams : kind != OR_UPDATE ? O.syms : O.upds;
    const int bn = kind == OR_UPDATE ? O.bn_upd : O.bn_sym;
    const uint32_t acc_full0 = or_smem(&S.acc_full[0]), acc_empty0 = or_smem(&S.acc_empty[0]);
    const int chunk = kind == OR_SQUARE && O.c == 0.0f ? 1 << 20 : 1;
    const uint32_t shift = or_buffers(O), buffers = 1u << shift;
    const int group0 = bn > 128 ? 2 * part : part;
    const uint32_t blk = ring + ORTHO_RING + (uint32_t)e * ORTHO_BLOCK;
    const uint32_t spare = bn == 64 ? blk + 4u * ORTHO_BLOCK : 0u;  // the other column part's
    const uint32_t taddr0 = S.tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(group0 * 64);
    bool ok = true;
    for (int64_t t = PAIR ? blockIdx.x >> 1 : blockIdx.x; ok && t < tiles; t += PAIR ? gridDim.x >> 1 : gridDim.x) {
        const OrthoTile T = or_tile<PAIR, SPLIT>(O, kind, t, rank);
        const int groups = min(bn > 128 ? 2 : 1, (T.width >> 6) - group0);
        const int chunks = (T.kblocks - 1) / chunk + 1;
        float v[128];
#pragma unroll
        for (int j = 0; j < 128; ++j) v[j] = 0.0f;
        for (int k = 0; k < chunks; ++k, ++acc) {
            const uint32_t b = acc & (buffers - 1u);
            ok = __all_sync(0xffffffffu, or_wait(acc_full0 + 8 * b, (acc >> shift) & 1u, &S.abort_flag));
            if (!ok) break;
            or_fence_after();
            if (groups > 0) {
#pragma unroll
                for (int j = 0; j < 64; j += 16) or_tmem_add16(taddr0 + b * (512u >> shift) + j, v + j);
            }
            if (groups > 1) {
#pragma unroll
                for (int j = 64; j < 128; j += 16) or_tmem_add16(taddr0 + b * (512u >> shift) + j, v + j);
            }
            or_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (PAIR) or_arrive_first<false>(acc_empty0 + 8 * b);
                else or_arrive(acc_empty0 + 8 * b);
            }
        }
        int m, n;
        if (O.list) m = O.list[T.which].m, n = O.list[T.which].n;
        else m = O.one.m, n = O.one.n;
        const int row = T.i * 128 + quad * 32 + lane;
        const int last_cb = or_b64(kind == OR_UPDATE ? n : m);  // a pair's tile may reach past the matrix
        // A split sum: every part to the workspace; the warp that comes last adds them in order and goes on
        if (SPLIT && ok && T.split > 1 && groups > 0 && !or_join(O, T, e, quad, group0, groups, lane, v)) continue;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const int cb = (T.c0 >> 6) + group0 + g;
            if (!ok || g >= groups || (PAIR && (cb >= last_cb || T.i >= or_mb(m)))) continue;
            if (kind == OR_UPDATE && step == O.steps - 1) or_finish_out(O, T.which, row, cb, blk, lane, v + 64 * g);
            else or_finish(O, kind, step, T.which, T.i, row, cb, blk, spare, lane, v + 64 * g);
        }
    }
    if (!ok) {
        if (lane == 0) atomicCAS(O.error, 0u, 3u);
        S.abort_flag = 1;
    }
    // the staging blocks' copies have been written before anyone reads them
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
}

// The steps' products: per step the Gram matrix, its polynomial and the update, a phase each over all
// matrices, each role running through the phases on its own.  PAIR: launched in clusters of two blocks, which
// work on tiles of 256 rows together (a block's own row block, half of the columns' operand each, the first
// block issuing), a third fewer bytes to fetch per product.
template <bool PAIR, bool SPLIT>
__global__ void __launch_bounds__(ORTHO_THREADS, 1) orthogonalize_kernel(const __grid_constant__ OrthoArgs O) {
    // the first kilobyte holds the barriers; the ring after it starts on the 1024 bytes of a swizzle atom
    extern __shared__ __align__(1024) unsigned char or_raw[];
    OrthoShared& S = *reinterpret_cast<OrthoShared*>(or_raw);
    static_assert(sizeof(OrthoShared) <= 1024, "shared state fits its kilobyte");
    const uint32_t ring = or_smem(or_raw) + 1024u;
    if (ring & 1023u) {  // never: dynamic shared memory alone starts on a kilobyte
        atomicCAS(O.error, 0u, 5u);
        return;
    }
    if (!O.x && *O.bad) return;  // the transition leaves everything as it was
    const int warp = threadIdx.x >> 5;
    const int rank = PAIR ? (int)or_cluster_rank() : 0;
    if (threadIdx.x == 0) {
        S.abort_flag = 0;
        for (int s = 0; s < ORTHO_STAGES; ++s) {
            or_mbar_init(or_smem(&S.full[s]), ORTHO_PRODUCERS);
            or_mbar_init(or_smem(&S.empty[s]), 1);
            or_mbar_init(or_smem(&S.peer[s]), 1);
        }
        for (int b = 0; b < 4; ++b) {
            or_mbar_init(or_smem(&S.acc_full[b]), 1);
            or_mbar_init(or_smem(&S.acc_empty[b]), PAIR ? 2 * ORTHO_EPI_WARPS : ORTHO_EPI_WARPS);
        }
        or_mbar_init(or_smem(&S.done), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x >= 128 && threadIdx.x < 256) {
        or_identity(O, or_raw + 1024 + ORTHO_RING + ORTHO_STAGING, threadIdx.x - 128, 8 * rank, or_square_back(O));  // of a pair each block has eight of its rows
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 0) {
        if (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(or_smem(&S.tmem)), "r"(512u)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(or_smem(&S.tmem)), "r"(512u)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    or_fence_before();
    __syncthreads();
    if (PAIR) or_cluster_sync();  // both blocks' barriers are there
    or_fence_after();
    const int phases = 3 * O.steps;
    uint32_t pipe = 0, acc = 0;
    if (warp == 0) {
        for (int p = 0; p < phases; ++p) {
            if (or_elect()) {
                if (PAIR && rank) or_relay(O, S, p % 3, pipe);
                else or_issue<PAIR, SPLIT>(O, S, ring, p % 3, pipe, acc);
            }
            __syncwarp();
            if (p + 1 < phases && !or_phase_end(O, S, p + 1)) break;
        }
    } else if (warp <= ORTHO_PRODUCERS) {
        for (int p = 0; p < phases; ++p) {
            if (or_elect()) or_produce<PAIR, SPLIT>(O, S, ring, p % 3, p / 3, rank, warp - 1, pipe);
            __syncwarp();
            if (p + 1 < phases && !or_phase_end(O, S, p + 1)) break;
        }
    } else {
        for (int p = 0; p < phases; ++p) {
            or_collect<PAIR, SPLIT>(O, S, ring, p % 3, p / 3, rank, warp - 1 - ORTHO_PRODUCERS, acc);
            if (p + 1 < phases && !or_phase_end(O, S, p + 1)) break;
        }
    }
    __syncthreads();
    if (warp == 0 && !(PAIR && rank)) {
        if (or_elect()) {
            // nothing that this thread issued is under way when the memory is freed
            or_commit<PAIR>(or_smem(&S.done));
            for (uint32_t i = 0; i < ORTHO_WAIT_TRIES && !or_try_wait(or_smem(&S.done), 0u); ++i) {
            }
        }
        __syncwarp();
    }
    if (PAIR) or_cluster_sync();  // neither block's shared memory or accumulators are in use any more
    if (warp == 0) {
        or_fence_after();
        if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(S.tmem), "r"(512u) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(S.tmem), "r"(512u) : "memory");
    }
}

// ------------------------------------------------------------ short sides up to 128

// A matrix whose short side is at most 128 stays in shared memory: a team of 1, 2, 4 or 8 blocks of a
// cluster holds up to three 64-column tiles of X each (long sides up to 1,536), and A and B whole.  A step
// is the team's Gram matrices of its columns, summed over the team (each block the rows that are its share,
// in rank order, and handed to all), the polynomial, which every block takes for itself, and the update of
// its own columns: no pass through L2 and no grid barrier, about a third of the time of the general path on
// a few such matrices.  A cluster is as large as the largest team; smaller teams share clusters and take
// part in all of the cluster's barriers.
constexpr int ORTHO_TEAM_TILES = 3;
constexpr int ORTHO_TEAM_MAX = 8;
constexpr int ORTHO_TEAM_THREADS = 512;                // warp 0 issues, warps 4 .. 15 take a row quarter of one column group each
constexpr int ORTHO_TEAM_A = 2 * ORTHO_TILE;           // A, then B: 128 x 128
constexpr int ORTHO_TEAM_SUM = 128 * 128 * 4;          // a block's own Gram matrix, fp32; then staging
constexpr int ORTHO_TEAM_SMEM = 1024 + ORTHO_TEAM_TILES * ORTHO_TILE + ORTHO_TEAM_A + ORTHO_TEAM_SUM + ORTHO_EYE;

struct OrthoTeam {
    uint64_t acc_full[2], acc_empty[2], done;
    double squares[ORTHO_TEAM_MAX];
    double part[ORTHO_TEAM_THREADS / 32];
    uint32_t tmem;
    volatile int abort_flag;
};

__device__ __forceinline__ uint32_t or_map(uint32_t addr, int rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    return a;
}

// 64 finished values of a row to a tile in shared memory, hi and lo
__device__ __forceinline__ void or_keep_rows(uint32_t tile, int row, const float* v) {
#pragma unroll
    for (int q = 0; q < 8; ++q) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float x0 = v[8 * q + 2 * j], x1 = v[8 * q + 2 * j + 1];
            const __half2 h = __floats2half2_rn(x0, x1);
            const float2 f = __half22float2(h);
            const __half2 l = __floats2half2_rn(x0 - f.x, x1 - f.y);
            hi[j] = *reinterpret_cast<const uint32_t*>(&h);
            lo[j] = *reinterpret_cast<const uint32_t*>(&l);
        }
        const uint32_t at = tile + (uint32_t)row * 128u + (uint32_t)((q ^ (row & 7)) << 4);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(hi[0]), "r"(hi[1]), "r"(hi[2]), "r"(hi[3]) : "memory");
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + 16384u), "r"(lo[0]), "r"(lo[1]), "r"(lo[2]), "r"(lo[3]) : "memory");
    }
}

// chunk q of a block's columns from a matrix's elements: lanes run along the stored rows
__device__ __forceinline__ void or_team_chunk(const OrthoArgs& O, const OrthoDesc& d, bool vector, int first, int q, const void* src,
                                              int type, float* u) {
    const int t = q >> 10, c = q & 1023;
    const int row = d.tall ? c & 127 : c >> 3, col = (first + t) * 64 + (d.tall ? c >> 7 : c & 7) * 8;
    const int live = row < d.m ? max(0, min(8, d.n - col)) : 0;
    if (d.tall) {
        const int64_t i = d.src + (int64_t)col * d.m + row;
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = e < live ? or_load(src, type, i + (int64_t)e * d.m) : 0.0f;
    } else {
        or_load8(src, type, d.src + (int64_t)row * d.n + col, vector, live, u);
    }
}

__global__ void __launch_bounds__(ORTHO_TEAM_THREADS, 1) orthogonalize_team_kernel(const __grid_constant__ OrthoArgs O, int cluster) {
    extern __shared__ __align__(1024) unsigned char or_raw[];
    OrthoTeam& S = *reinterpret_cast<OrthoTeam*>(or_raw);
    static_assert(sizeof(OrthoTeam) <= 1024, "shared state fits its kilobyte");
    const uint32_t xs = or_smem(or_raw) + 1024u;
    const uint32_t as = xs + ORTHO_TEAM_TILES * ORTHO_TILE, sums = as + ORTHO_TEAM_A, eye_at = sums + ORTHO_TEAM_SUM;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (xs & 1023u) {  // never: dynamic shared memory alone starts on a kilobyte
        atomicCAS(O.error, 0u, 5u);
        return;
    }
    if (!O.x && *O.bad) {  // the transition leaves everything as it was but the gradients
        if (blockIdx.x < O.slots) {
            const OrthoDesc d = or_get(O, or_find(O, blockIdx.x, &OrthoDesc::slot0, O.one.team));
            const int64_t total = (int64_t)d.m * d.n;
            for (int64_t i = (int64_t)(blockIdx.x - d.slot0) * ORTHO_TEAM_THREADS + threadIdx.x; i < total; i += (int64_t)d.team * ORTHO_TEAM_THREADS)
                O.grad[d.src + i] = 0.0f;
        }
        return;
    }
    const bool here = blockIdx.x < O.slots;  // the last cluster may have blocks to spare
    OrthoDesc d = {};
    int which = 0, rank = 0;
    if (here) {
        which = (int)or_find(O, blockIdx.x, &OrthoDesc::slot0, O.one.team);
        d = or_get(O, which);
        rank = (int)(blockIdx.x - d.slot0);
    } else {
        d.team = 1;
    }
    const int nb = or_b64(d.n), m64 = or_b64(d.m), team = d.team;
    const int each = (nb + team - 1) / team;                        // tiles of a block
    const int first = rank * each;                                  // its first column block
    const int tiles = max(0, min(each, nb - first));
    const int base = cluster > 1 ? (int)or_cluster_rank() - rank : 0;  // the team's first block in the cluster

    if (threadIdx.x == 0) {
        S.abort_flag = 0;
        for (int b = 0; b < 2; ++b) {
            or_mbar_init(or_smem(&S.acc_full[b]), 1);
            or_mbar_init(or_smem(&S.acc_empty[b]), ORTHO_TEAM_THREADS / 32 - 4);
        }
        or_mbar_init(or_smem(&S.done), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x >= 128 && threadIdx.x < 256) {
        or_identity(O, or_raw + (eye_at - or_smem(or_raw)), threadIdx.x - 128, 0, or_back(d.m));
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(or_smem(&S.tmem)), "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }

    // ---------------------------------------------------- the direction, its norm, and X
    const OrthoDirection k = or_controls(O);
    const bool vector = O.aligned && d.src % 4 == 0 && d.n % 4 == 0;
    // Chunks of 8 columns, rolled loops; the squares' pass leaves the values in L1 and L2 for the second.
    const int chunks_all = tiles * 1024;
    double total = 0.0;
    if (O.x) {
        double square = 0.0;
#pragma unroll 2
        for (int q = threadIdx.x; q < chunks_all; q += ORTHO_TEAM_THREADS) {
            float u[8];
            or_team_chunk(O, d, vector, first, q, O.x, O.x_type, u);
#pragma unroll
            for (int e = 0; e < 8; ++e) square += (double)u[e] * (double)u[e];
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) square += __shfl_xor_sync(0xffffffffu, square, o);
        if (lane == 0) S.part[warp] = square;
        if (cluster > 1) or_cluster_sync();  // the others run: their shared memory may be written
        else __syncthreads();
        if (threadIdx.x < team) {
            double own = 0.0;
            for (int w = 0; w < ORTHO_TEAM_THREADS / 32; ++w) own += S.part[w];
            const uint32_t at = or_smem(&S.squares[rank]);
            if (team == 1) S.squares[0] = own;
            else asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(or_map(at, base + (int)threadIdx.x)), "d"(own) : "memory");
        }
        if (cluster > 1) or_cluster_sync();
        else __syncthreads();
        for (int r = 0; r < team; ++r) total += S.squares[r];
    } else {
        if (cluster > 1) or_cluster_sync();
        const int64_t spans = ((int64_t)d.m * d.n + ORTHO_SPAN - 1) / ORTHO_SPAN;
        for (int64_t r = 0; r < spans; ++r) total += __ldg(O.sums + d.span0 + r);
    }
    const double wide = or_wide(O, total);
    const float scale = (float)wide;
    const bool plain = scale < 1.0e30f;
#pragma unroll 2
    for (int q = threadIdx.x; q < chunks_all; q += ORTHO_TEAM_THREADS) {
        float u[8], m[8];
        or_team_chunk(O, d, vector, first, q, O.x ? O.x : O.grad, O.x ? O.x_type : 0, u);
        const int t = q >> 10, c = q & 1023;
        const int row = d.tall ? c & 127 : c >> 3, chunk = d.tall ? c >> 7 : c & 7, col = (first + t) * 64 + chunk * 8;
        const int live = row < d.m ? max(0, min(8, d.n - col)) : 0;
        if (!O.x) {
            or_team_chunk(O, d, vector, first, q, O.momentum, 0, m);
            const int64_t i = d.src + (d.tall ? (int64_t)col * d.m + row : (int64_t)row * d.n + col);
            const int64_t next = d.tall ? d.m : 1;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                m[e] = or_momentum(k, u[e], m[e]);
                u[e] = or_direction(k, u[e], m[e]);
                if (e < live) O.momentum[i + e * next] = m[e];
            }
        }
        __align__(16) __half hi[8];
        __align__(16) __half lo[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) or_split(e < live ? (plain ? u[e] * scale : (float)((double)u[e] * wide)) : 0.0f, hi[e], lo[e]);
        unsigned char* at = or_raw + 1024 + t * ORTHO_TILE + row * 128 + ((chunk ^ (row & 7)) << 4);
        *reinterpret_cast<uint4*>(at) = *reinterpret_cast<uint4*>(hi);
        *reinterpret_cast<uint4*>(at + 16384) = *reinterpret_cast<uint4*>(lo);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    or_fence_before();
    __syncthreads();
    or_fence_after();

    // ---------------------------------------------------- the steps
    const uint32_t acc_full0 = or_smem(&S.acc_full[0]), acc_empty0 = or_smem(&S.acc_empty[0]);
    const uint32_t tmem = S.tmem;
    const int e = warp - 4, quad = warp & 3, part = e >> 2;  // epilogue warps: column group `part`
    const int row = quad * 32 + lane;
    uint32_t acc = 0;
    for (int step = 0; step < O.steps; ++step) {
        for (int kind = 0; kind < 3; ++kind) {
            const bool linear = kind == OR_SQUARE && O.c == 0.0f;
            const int kblocks = tiles == 0 && kind != OR_SQUARE ? 0 : kind == OR_GRAM ? tiles : m64;
            const int groups_all = kind == OR_UPDATE ? tiles : m64;  // 64-column groups of the product
            float v[64];
#pragma unroll
            for (int j = 0; j < 64; ++j) v[j] = 0.0f;
            const bool mine = part < groups_all;
            bool ok = true;
            if (warp == 0) {
                if (or_elect()) {
                    const uint32_t idesc = or_idesc<false>(groups_all * 64, kind == OR_UPDATE), eye_idesc = or_idesc<false>(16, 0);
                    const uint32_t eye = or_desc(eye_at, 16);
                    for (int kb = 0; kb < kblocks; ++kb) {
                        // K-major operands: column block kb of X or A against the same rows; the update: column
                        // block kb of B against rows 64 kb of X, its column blocks a tile apart
                        const uint32_t b = acc & 1u;
                        if (!linear || kb == 0) {
                            if (!or_wait(acc_empty0 + 8 * b, ((acc >> 1) & 1u) ^ 1u, &S.abort_flag)) {
                                ok = false;
                                break;
                            }
                            or_fence_after();
                        }
                        const uint32_t dd = tmem + b * 256u;
                        const uint32_t at = (kind == OR_GRAM ? xs : as) + (uint32_t)kb * ORTHO_TILE;
                        const uint32_t a = or_desc(at, 16), al = a + (16384u >> 4);
                        const uint32_t bh = kind == OR_UPDATE ? or_desc(xs + (uint32_t)kb * 8192u, ORTHO_TILE) : a;
                        const uint32_t bl = bh + (16384u >> 4), b_step = kind == OR_UPDATE ? 2048u >> 4 : 2u;
                        const uint32_t dc = dd + (uint32_t)kb * 64u;
                        if (linear) {
#pragma unroll
                            for (int ks = 0; ks < 4; ++ks) {
                                or_mma<false>(dc + ks * 16, al + ks * 2, eye, eye_idesc, 0u);
                                or_mma<false>(dc + ks * 16, a + ks * 2, eye, eye_idesc, 1u);
                            }
                        } else {
#pragma unroll
                            for (int ks = 0; ks < 4; ++ks) or_mma<false>(dd, al + ks * 2, bh + ks * b_step, idesc, ks > 0);
#pragma unroll
                            for (int ks = 0; ks < 4; ++ks) or_mma<false>(dd, a + ks * 2, bl + ks * b_step, idesc, 1u);
                            if (kind == OR_SQUARE) {
#pragma unroll
                                for (int ks = 0; ks < 4; ++ks) or_identity_small<false>(dc + ks * 16, a + ks * 2, al + ks * 2, eye, eye_idesc);
                            }
#pragma unroll
                            for (int ks = 0; ks < 4; ++ks) or_mma<false>(dd, a + ks * 2, bh + ks * b_step, idesc, 1u);
                            if (kind == OR_SQUARE) {
#pragma unroll
                                for (int ks = 0; ks < 4; ++ks) or_mma<false>(dc + ks * 16, a + ks * 2, eye, eye_idesc, 1u);
                            }
                        }
                        if (!linear || kb == kblocks - 1) {
                            or_commit<false>(acc_full0 + 8 * b);
                            ++acc;
                        }
                    }
                    if (!ok) {
                        atomicCAS(O.error, 0u, 2u);
                        S.abort_flag = 1;
                    }
                }
                __syncwarp();
            } else if (e >= 0) {
                const int chunks = linear ? (kblocks > 0) : kblocks;
                const uint32_t taddr0 = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(part * 64);
                for (int c = 0; c < chunks; ++c, ++acc) {
                    const uint32_t b = acc & 1u;
                    ok = __all_sync(0xffffffffu, or_wait(acc_full0 + 8 * b, (acc >> 1) & 1u, &S.abort_flag));
                    if (!ok) break;
                    or_fence_after();
                    if (mine) {
#pragma unroll
                        for (int j = 0; j < 64; j += 16) or_tmem_add16(taddr0 + b * 256u + j, v + j);
                    }
                    or_fence_before();
                    __syncwarp();
                    if (lane == 0) or_arrive(acc_empty0 + 8 * b);
                }
                if (!ok) {
                    if (lane == 0) atomicCAS(O.error, 0u, 3u);
                    S.abort_flag = 1;
                }
                if (kind == OR_GRAM) {
#pragma unroll
                    for (int j = 0; j < 64; ++j) v[j] *= or_back(d.n) * (ORTHO_SA / (ORTHO_SX * ORTHO_SX));
                    if (team == 1) {
                        if (mine) or_keep_rows(as + part * ORTHO_TILE, row, v);
                    } else if (part < m64) {
                        // to the block whose share this row is: [rank][its rows][32 chunks of four columns],
                        // chunks swizzled by the row
                        const int rows = 128 / team;
                        const uint32_t there = or_map(sums, base + row / rows) + (uint32_t)(rank * rows + row % rows) * 512u;
#pragma unroll
                        for (int q = 0; q < 16; ++q)
                            asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(there + (uint32_t)(((part * 16 + q) ^ lane) << 4)),
                                         "f"(v[4 * q]), "f"(v[4 * q + 1]), "f"(v[4 * q + 2]), "f"(v[4 * q + 3])
                                         : "memory");
                    }
                } else if (kind == OR_SQUARE) {
                    const float factor = or_square_factor(O, or_back(d.m)) * (ORTHO_SB / (ORTHO_SA * ORTHO_SA)), diagonal = O.a * ORTHO_SB;
                    if (mine) {
#pragma unroll
                        for (int j = 0; j < 64; ++j) v[j] = fmaf(v[j], factor, row == part * 64 + j ? diagonal : 0.0f);
                        or_keep_rows(as + part * ORTHO_TILE, row, v);
                    }
                } else if (mine && ok) {
                    if (step + 1 < O.steps) {
#pragma unroll
                        for (int j = 0; j < 64; ++j) v[j] *= 1.0f / ORTHO_SB;
                        or_keep_rows(xs + part * ORTHO_TILE, row, v);
                    } else {
                        or_finish_out(O, which, row, first + part, sums + (uint32_t)e * ORTHO_BLOCK, lane, v);
                    }
                }
            }
            __syncwarp();
            if (kind == OR_GRAM && cluster > 1) {
                or_cluster_sync();
                if (team > 1) {
                    // this block's rows, summed over the team in rank order, as pairs to every block of the team
                    const int rows = 128 / team;
                    for (int q = threadIdx.x; q < rows * 32; q += ORTHO_TEAM_THREADS) {
                        const int r = rank * rows + (q >> 5), chunk = q & 31;  // four columns
                        if (chunk >= m64 * 16) continue;
                        float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        for (int j = 0; j < team; ++j) {
                            float4 t;
                            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                                         : "=f"(t.x), "=f"(t.y), "=f"(t.z), "=f"(t.w)
                                         : "r"(sums + (uint32_t)(j * rows + (q >> 5)) * 512u + (uint32_t)((chunk ^ (r & 31)) << 4))
                                         : "memory");
                            f.x += t.x, f.y += t.y, f.z += t.z, f.w += t.w;
                        }
                        const __half2 h0 = __floats2half2_rn(f.x, f.y), h1 = __floats2half2_rn(f.z, f.w);
                        const float2 g0 = __half22float2(h0), g1 = __half22float2(h1);
                        const __half2 l0 = __floats2half2_rn(f.x - g0.x, f.y - g0.y), l1 = __floats2half2_rn(f.z - g1.x, f.w - g1.y);
                        // eight bytes of a 16-byte chunk of tile chunk / 16
                        const uint32_t to = as + (uint32_t)(chunk >> 4) * ORTHO_TILE + (uint32_t)r * 128u +
                                            (uint32_t)((((chunk & 15) >> 1) ^ (r & 7)) << 4) + (uint32_t)(chunk & 1) * 8u;
                        for (int j = 0; j < team; ++j) {
                            const uint32_t there = or_map(to, base + j);
                            asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(there),
                                         "r"(*reinterpret_cast<const uint32_t*>(&h0)), "r"(*reinterpret_cast<const uint32_t*>(&h1))
                                         : "memory");
                            asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(there + 16384u),
                                         "r"(*reinterpret_cast<const uint32_t*>(&l0)), "r"(*reinterpret_cast<const uint32_t*>(&l1))
                                         : "memory");
                        }
                    }
                    asm volatile("fence.proxy.async;" ::: "memory");
                    __syncwarp();
                }
                or_cluster_sync();
                asm volatile("fence.proxy.async;" ::: "memory");
                or_fence_after();
            } else {
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                or_fence_before();
                __syncthreads();
                or_fence_after();
            }
        }
    }
    if (warp == 0) {
        if (or_elect()) {
            or_commit<false>(or_smem(&S.done));
            for (uint32_t i = 0; i < ORTHO_WAIT_TRIES && !or_try_wait(or_smem(&S.done), 0u); ++i) {
            }
        }
        __syncwarp();
        or_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// ------------------------------------------------------------ host

constexpr int64_t ORTHO_BUDGET = 1ll << 30;  // bytes of tiles that one launch works in, where a matrix alone does not need more

// blocks of a matrix's team, 0 where it takes the general path
static int or_team(int m, int n) {
    if (m > 128 || or_b64(n) > ORTHO_TEAM_MAX * ORTHO_TEAM_TILES) return 0;
    int team = 1;
    while (team * ORTHO_TEAM_TILES < or_b64(n)) team *= 2;
    return team;
}
static int64_t or_tiles_bytes(int m, int n) { return or_team(m, n) ? 0 : 2 * or_x_bytes(m, n) + 2 * or_a_bytes(m); }
static int64_t or_spans(int64_t total) { return (total + ORTHO_SPAN - 1) / ORTHO_SPAN; }
static int64_t or_syms(int m, int bn, int pair, int mirror) {
    int64_t n = 0;
    for (int i = 0; i < or_row_blocks(m, pair); ++i) n += or_sym_row(m, i, bn, pair, mirror);
    return n;
}
static int64_t or_upds(int m, int n, int bn, int pair) {
    return (int64_t)or_row_blocks(m, pair) * ((or_b64(n) * 64 + bn - 1) / bn);
}

static OrthoDesc or_make(int64_t rows, int64_t cols) {
    OrthoDesc d = {};
    d.tall = rows > cols;
    d.m = (int)(d.tall ? cols : rows);
    d.n = (int)(d.tall ? rows : cols);
    d.adjust = 1.0f;
    d.team = or_team(d.m, d.n);
    return d;
}

// Output tile shapes: those whose busiest block has least to do, the tiles being dealt out in turn.  A k-block
// of 64 and an output tile's end cost (microseconds) what they were measured to on matrices of 4,096 and of
// 256 x 16,384, for tiles of 128 x 64, x 128, x 192 and x 256 by one block and of 256 x 256 by a pair, and
// OR_MIRROR more where a tile's mirror image is written too.  Wide tiles fetch less per multiply-add, narrow
// ones spread a few small matrices over more SMs; small matrices have SMs to spare for both triangles.
//
// A Gram matrix has few tiles, and each sums over the whole long side: where few matrices have long ones,
// several blocks (not pairs) sum parts of it, and the last of them adds the parts (OR_JOIN, and OR_PART per part and
// group of 64 columns of a warp: loads of few registers each, one L2 latency after the other).  The kernel that can do this takes 4 % longer where
// it has nothing to split, so a split has to save a tenth of the estimate.  Five steps of 256 x 16,384 take
// 373 us (whole sums 935), of 256 x 2,048 208 (226), of 200 x 5,000 253 (376).
static const int OR_SHAPES = 5;
static const int OR_WIDTHS[OR_SHAPES] = {64, 128, 192, 256, 256};
static const double OR_BLOCK[OR_SHAPES] = {0.64, 0.88, 1.1, 1.27, 1.18}, OR_END[OR_SHAPES] = {2.6, 3.2, 4.2, 4.5, 4.5};
static const double OR_MIRROR = 2.5, OR_JOIN = 3.0, OR_PART = 2.0;
static const int OR_SPLIT = 16, OR_SPLIT_BLOCKS = 4;  // most parts, fewest k-blocks of one

struct OrthoShape {
    int bn_sym, bn_upd, pair, mirror;
    double target;  // of a Gram matrix's item, from which its parts follow; 0: whole
};
static double or_cost(int kind, int m, int n, int w, int mirror, int split) {
    const double end = OR_END[w] + (kind != OR_UPDATE && mirror && m > (w == 4 ? 256 : 128) ? OR_MIRROR : 0.0);
    const double sum = or_b64(kind == OR_GRAM ? n : m) * OR_BLOCK[w];
    return end + (split > 1 ? (sum / split) * 1.04 + OR_JOIN + OR_PART * (w < 2 ? 1 : 2) * split : sum);
}
// parts of a Gram matrix's sums: the fewest that bring an item's time down to `target`, or its least time's
static int or_split(int m, int n, int w, int mirror, double target) {
    int best = 1, most = or_b64(n) / OR_SPLIT_BLOCKS;
    double least = or_cost(OR_GRAM, m, n, w, mirror, 1);
    if (target <= 0.0) return 1;
    for (int split = 2; least > target && split <= OR_SPLIT && split <= most; ++split) {
        const double t = or_cost(OR_GRAM, m, n, w, mirror, split);
        if (t < least) least = t, best = split;
    }
    return best;
}
// `count` matrices of list, or of one size
static OrthoShape or_choose(const OrthoDesc* list, int64_t count, bool same) {
    const int sms = sm_count() < 1024 ? sm_count() : 1024;
    OrthoShape best = {64, 64, 0, 1, 0.0};
    double least = -1.0, load[1024];
    for (int pass = 0; pass < 3; ++pass) {  // single blocks, pairs, single blocks that split sums
        const int pair = pass == 1, blocks = pair ? sms / 2 : sms, w0 = pair ? 4 : 0, w1 = pair ? 5 : 4;
        // the busiest block's time of a kind of product
        auto busiest = [&](int kind, int w, int mirror, double target) {
            double top = 0.0;
            int at = 0;
            for (int b = 0; b < blocks; ++b) load[b] = 0.0;
            for (int64_t i = 0; i < (same ? 1 : count); ++i) {
                const int m = list[i].m, n = list[i].n, split = kind == OR_GRAM ? or_split(m, n, w, mirror, target) : 1;
                const double c = or_cost(kind, m, n, w, mirror, split);
                const int64_t tiles =
                    split * (kind == OR_UPDATE ? or_upds(m, n, OR_WIDTHS[w], pair) : or_syms(m, OR_WIDTHS[w], pair, mirror));
                if (same) return (double)((count * tiles + blocks - 1) / blocks) * c;
                for (int64_t t = tiles; t > 0; --t) {
                    load[at] += c;
                    if (load[at] > top) top = load[at];
                    if (++at == blocks) at = 0;
                }
            }
            return top;
        };
        double sym = -1.0, upd = -1.0;
        OrthoShape shape = {0, 0, pair, 1, 0.0};
        for (int w = w0; w < w1; ++w) {
            for (int mirror = 0; mirror < 2; ++mirror) {
                const double square = busiest(OR_SQUARE, w, mirror, 0.0), whole = busiest(OR_GRAM, w, mirror, 0.0);
                // a split's items: a half of the busiest block's time at whole sums, a quarter and so on
                for (int i = pass == 2 ? 1 : 0; i < (pass == 2 ? 5 : 1); ++i) {
                    const double target = i ? whole / (1 << i) : 0.0, t = square + (i ? busiest(OR_GRAM, w, mirror, target) : whole);
                    if (sym < 0.0 || t < sym) sym = t, shape.bn_sym = OR_WIDTHS[w], shape.mirror = mirror, shape.target = target;
                }
            }
            const double t = busiest(OR_UPDATE, w, 0, 0.0);
            if (upd < 0.0 || t < upd) upd = t, shape.bn_upd = OR_WIDTHS[w];
        }
        if (least < 0.0 || sym + upd < (pass == 2 ? 0.9 : 1.0) * least) least = sym + upd, best = shape;
    }
    return best;
}
static int or_split_of(int m, int n, const OrthoShape& s) {
    int w = 0;
    while (OR_WIDTHS[w] != s.bn_sym) ++w;
    return or_split(m, n, w, s.mirror, s.target);
}
// bytes of the parts and arrival counters of `items` split items
static int64_t or_parts_bytes(int64_t items, const OrthoShape& s) { return items * 128 * s.bn_sym * 4; }
static int64_t or_arrived_bytes(int64_t items) { return items * ORTHO_EPI_WARPS * 4; }

static int64_t or_up(int64_t v) { return (v + 1023) / 1024 * 1024; }

static int or_squares(const OrthoArgs& O, cudaStream_t s) {
    PBG_REQUIRE(O.spans < (1ll << 31), "orthogonalize: too many elements for one launch");
    orthogonalize_squares_kernel<<<(unsigned)O.spans, ORTHO_FLAT, 0, s>>>(O);
    return launch_status("orthogonalize: squares");
}

// the matrices with teams: O.list (largest teams first) or O.one, O.slots blocks
static int or_teams(const OrthoArgs& O, int cluster, cudaStream_t s) {
    static int configured[64] = {0};
    int dev = 0, rc = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        rc = cuda_status(cudaFuncSetAttribute(orthogonalize_team_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, ORTHO_TEAM_SMEM),
                         "orthogonalize: shared memory size");
        if (rc) return rc;
        if (dev >= 0 && dev < 64) configured[dev] = 1;
    }
    const int64_t grid = (O.slots + cluster - 1) / cluster * cluster;
    PBG_REQUIRE(grid < (1ll << 31), "orthogonalize: too many matrices for one launch");
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)grid);
    config.blockDim = dim3(ORTHO_TEAM_THREADS);
    config.dynamicSmemBytes = ORTHO_TEAM_SMEM;
    config.stream = s;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeClusterDimension;
    attribute[0].val.clusterDim.x = cluster;
    attribute[0].val.clusterDim.y = attribute[0].val.clusterDim.z = 1;
    config.attrs = attribute;
    config.numAttrs = cluster > 1 ? 1 : 0;
    void* args[] = {const_cast<OrthoArgs*>(&O), &cluster};
    return cuda_status(cudaLaunchKernelExC(&config, (const void*)orthogonalize_team_kernel, args), "orthogonalize: team launch");
}

// conversion, then the products
static int or_products(const OrthoArgs& O, int64_t arrived_bytes, cudaStream_t s) {
    const void* const kernels[3] = {(const void*)orthogonalize_kernel<false, false>, (const void*)orthogonalize_kernel<true, false>,
                                    (const void*)orthogonalize_kernel<false, true>};
    static int pairs_at_once[64] = {0};  // pairs of blocks that the device runs at once, from the first call on
    int dev = 0, rc = 0;
    rc = cuda_status(cudaGetDevice(&dev), "orthogonalize: device");
    if (rc) return rc;
    PBG_REQUIRE(dev < 64, "orthogonalize: at most 64 devices");
    if (!pairs_at_once[dev]) {
        for (int i = 0; i < 3; ++i) {
            rc = cuda_status(cudaFuncSetAttribute(kernels[i], cudaFuncAttributeMaxDynamicSharedMemorySize, ORTHO_SMEM),
                             "orthogonalize: shared memory size");
            if (rc) return rc;
        }
        cudaLaunchConfig_t config = {};
        config.gridDim = dim3((unsigned)sm_count() / 2 * 2), config.blockDim = dim3(ORTHO_THREADS);
        config.dynamicSmemBytes = ORTHO_SMEM;
        cudaLaunchAttribute cluster[1];
        cluster[0].id = cudaLaunchAttributeClusterDimension;
        cluster[0].val.clusterDim.x = 2;
        cluster[0].val.clusterDim.y = cluster[0].val.clusterDim.z = 1;
        config.attrs = cluster, config.numAttrs = 1;
        int pairs = 0;
        rc = cuda_status(cudaOccupancyMaxActiveClusters(&pairs, kernels[1], &config), "orthogonalize: pairs of blocks");
        if (rc) return rc;
        PBG_REQUIRE(pairs >= 1, "orthogonalize: the device runs no pair of blocks");
        pairs_at_once[dev] = pairs;
    }
    // the barrier's word and, behind it, the split sums' arrivals
    rc = cuda_status(cudaMemsetAsync(O.barrier, 0, (size_t)(256 + arrived_bytes), s), "orthogonalize: barrier");
    if (rc) return rc;
    PBG_REQUIRE(O.convs < (1ll << 31), "orthogonalize: too many tiles for one launch");
    orthogonalize_convert_kernel<<<(unsigned)O.convs, ORTHO_FLAT, 0, s>>>(O);
    rc = launch_status("orthogonalize: conversion");
    if (rc) return rc;
    // one block per SM, all of them running at once
    int64_t tiles = O.syms > O.upds ? O.syms : O.upds;
    if (O.grams > tiles) tiles = O.grams;
    const int64_t most = O.pair ? std::min(sm_count() / 2, pairs_at_once[dev]) * 2 : sm_count();
    const int64_t want = O.pair ? 2 * tiles : tiles;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)(want < most ? want : most));
    config.blockDim = dim3(ORTHO_THREADS);
    config.dynamicSmemBytes = ORTHO_SMEM;
    config.stream = s;
    cudaLaunchAttribute attribute[2];
    attribute[0].id = cudaLaunchAttributeCooperative;
    attribute[0].val.cooperative = 1;
    attribute[1].id = cudaLaunchAttributeClusterDimension;
    attribute[1].val.clusterDim.x = 2;
    attribute[1].val.clusterDim.y = attribute[1].val.clusterDim.z = 1;
    config.attrs = attribute;
    config.numAttrs = O.pair ? 2 : 1;
    void* args[] = {const_cast<OrthoArgs*>(&O)};
    return cuda_status(cudaLaunchKernelExC(&config, kernels[O.pair ? 1 : O.grams > O.syms ? 2 : 0], args),
                       "orthogonalize: cooperative launch");
}

// The fp16 scales hold while no singular value passes 2 and |a + b s^2 + c s^4| stays below 15: the range
// [0, 1] of the first iterate followed step by step, the extremes of s (a + b s^2 + c s^4) and of its factor
// being at the ends of a range and where their derivatives vanish (the polynomials in use stay within 1.3
// and 3.5).
static int or_check_polynomial(int steps, float a, float b, float c) {
    PBG_REQUIRE(steps >= 1 && steps <= 100, "orthogonalize: steps must be in [1,100]");
    PBG_REQUIRE(c == 0.0f || (b / c < 7.9f && b / c > -7.9f), "orthogonalize: |b| must be below 7.9 |c| where c is not 0");
    const double A = a, B = b, C = c;
    double at[4] = {0.0, -1.0, -1.0, -1.0};  // squares of the inner extremes' places; the range's end joins them
    if (C != 0.0) {
        const double disc = 9.0 * B * B - 20.0 * A * C;
        if (disc >= 0.0) at[1] = (-3.0 * B + sqrt(disc)) / (10.0 * C), at[2] = (-3.0 * B - sqrt(disc)) / (10.0 * C);
        at[3] = -B / (2.0 * C);
    } else if (B != 0.0) {
        at[1] = -A / (3.0 * B);
    }
    double top = 1.0;
    for (int k = 0; k < steps; ++k) {
        double next = 0.0;
        for (int i = 0; i < 5; ++i) {
            const double g = i < 4 ? at[i] : top * top;
            if (!(g >= 0.0 && g <= top * top) && i < 4) continue;
            const double q = fabs(A + g * (B + g * C));
            PBG_REQUIRE(q < 15.0, "orthogonalize: the coefficients leave the range of the products");
            next = fmax(next, sqrt(g) * q);
        }
        PBG_REQUIRE(next < 1.9, "orthogonalize: the coefficients let singular values grow past 2");
        if (next <= top && k > 0) break;
        top = fmax(next, 1.0);
    }
    return 0;
}

static int64_t or_at_once(int64_t batch, int m, int n) {
    if (or_team(m, n)) return batch;
    int64_t k = ORTHO_BUDGET / or_tiles_bytes(m, n);
    k = k < 1 ? 1 : k;
    return k < batch ? k : batch;
}

// a stack of matrices of one size: how many a launch takes, its tiles' shape, and the workspace
struct OrthoUniform {
    int64_t at_once, sums, parts, tiles, bytes;
    OrthoShape shape;
    int split;
};
static OrthoUniform or_uniform(int64_t batch, const OrthoDesc& d) {
    OrthoUniform U;
    U.at_once = or_at_once(batch, d.m, d.n);
    U.shape = or_choose(&d, U.at_once, true);
    U.split = or_split_of(d.m, d.n, U.shape);
    const int64_t items = U.split > 1 ? U.at_once * U.split * or_syms(d.m, U.shape.bn_sym, U.shape.pair, U.shape.mirror) : 0;
    U.sums = or_up(256 + or_arrived_bytes(items));
    U.parts = U.sums + or_up(U.at_once * or_spans((int64_t)d.m * d.n) * 8);
    U.tiles = U.parts + or_up(or_parts_bytes(items, U.shape));
    U.bytes = U.tiles + U.at_once * or_tiles_bytes(d.m, d.n);
    return U;
}

}  // namespace pbg

using namespace pbg;

extern "C" {

int64_t pbg_orthogonalize_workspace(int64_t batch, int64_t rows, int64_t cols) {
    if (batch <= 0 || rows <= 0 || cols <= 0 || rows > 65536 || cols > 65536) return 0;
    const OrthoDesc d = or_make(rows, cols);
    if (d.team) return 1024;
    return or_uniform(batch, d).bytes;
}

int pbg_orthogonalize(int64_t batch, int64_t rows, int64_t cols, const void* x, int32_t x_type, void* out, int32_t out_type,
                      int32_t steps, float a, float b, float c, double eps, void* workspace, int64_t workspace_bytes,
                      uint32_t* error, void* stream) {
    PBG_REQUIRE(batch >= 0 && rows >= 0 && cols >= 0, "orthogonalize: negative size");
    PBG_REQUIRE(rows <= 65536 && cols <= 65536, "orthogonalize: at most 65,536 rows and columns");
    PBG_REQUIRE(x_type >= 0 && x_type <= 2 && out_type >= 0 && out_type <= 2, "orthogonalize: unknown type");
    PBG_REQUIRE(eps >= 0.0, "orthogonalize: epsilon must not be negative");
    int rc = or_check_polynomial(steps, a, b, c);
    if (rc) return rc;
    if (batch == 0 || rows == 0 || cols == 0) return 0;
    PBG_REQUIRE(x && out && workspace && error, "orthogonalize: null pointer");
    PBG_REQUIRE((uintptr_t)workspace % 256 == 0, "orthogonalize: workspace must be 256-byte aligned");
    OrthoArgs O = {};
    O.one = or_make(rows, cols);
    const int m = O.one.m, n = O.one.n;
    O.one_src = rows * cols;
    O.steps = steps, O.a = a, O.b = b, O.c = c, O.eps = eps;
    O.x_type = x_type, O.out_type = out_type, O.error = error;
    if (O.one.team) {
        PBG_REQUIRE(workspace_bytes >= 1024, "orthogonalize: workspace too small");
        O.count = batch, O.slots = batch * O.one.team;
        O.x = x, O.out = out;
        O.aligned = (uintptr_t)x % 16 == 0 && (uintptr_t)out % 16 == 0;
        return or_teams(O, O.one.team, as_stream(stream));
    }
    const OrthoUniform U = or_uniform(batch, O.one);
    PBG_REQUIRE(workspace_bytes >= U.bytes, "orthogonalize: workspace too small");
    unsigned char* w = static_cast<unsigned char*>(workspace);
    O.barrier = reinterpret_cast<uint32_t*>(w);
    O.arrived = reinterpret_cast<uint32_t*>(w + 256);
    O.sums = reinterpret_cast<double*>(w + U.sums);
    O.parts = reinterpret_cast<float*>(w + U.parts);
    O.tiles = w + U.tiles;
    O.bn_sym = U.shape.bn_sym, O.bn_upd = U.shape.bn_upd, O.pair = U.shape.pair, O.mirror = U.shape.mirror;
    O.one.split = U.split;
    O.one_ws = or_tiles_bytes(m, n);
    O.one_span = or_spans(rows * cols);
    O.one_conv = (int64_t)or_mb(m) * or_b64(n);
    O.one_sym = or_syms(m, O.bn_sym, O.pair, O.mirror), O.one_upd = or_upds(m, n, O.bn_upd, O.pair);
    O.one_gram = O.one_sym * U.split;
    const int64_t xs = x_type == 0 ? 4 : 2, os = out_type == 0 ? 4 : 2;
    for (int64_t at = 0; at < batch; at += U.at_once) {
        O.count = batch - at < U.at_once ? batch - at : U.at_once;
        O.spans = O.count * O.one_span, O.convs = O.count * O.one_conv;
        O.grams = O.count * O.one_gram, O.syms = O.count * O.one_sym, O.upds = O.count * O.one_upd;
        O.x = static_cast<const unsigned char*>(x) + at * rows * cols * xs;
        O.out = static_cast<unsigned char*>(out) + at * rows * cols * os;
        O.aligned = (uintptr_t)O.x % 16 == 0 && (uintptr_t)O.out % 16 == 0;
        rc = or_squares(O, as_stream(stream));
        if (!rc) rc = or_products(O, U.split > 1 ? or_arrived_bytes(O.grams) : 0, as_stream(stream));
        if (rc) return rc;
    }
    return 0;
}

int64_t pbg_muon_descriptor_bytes(void) { return (int64_t)sizeof(OrthoDesc); }

int64_t pbg_muon_plan_words(int64_t count) { return count < 0 ? 0 : 10 + 7 * count; }

int pbg_muon_plan(int64_t count, const int64_t* offset, const int64_t* rows, const int64_t* cols, const float* adjust,
                  void* descriptors, int64_t* plan) {
    PBG_REQUIRE(count >= 1 && offset && rows && cols && adjust && descriptors && plan, "muon_plan: null argument");
    OrthoDesc* list = static_cast<OrthoDesc*>(descriptors);
    for (int64_t i = 0; i < count; ++i) {
        PBG_REQUIRE(offset[i] >= 0 && rows[i] >= 1 && cols[i] >= 1 && rows[i] <= 65536 && cols[i] <= 65536,
                    "muon_plan: matrix %lld: sizes must be in [1,65536]", (long long)i);
        list[i] = or_make(rows[i], cols[i]);
        list[i].src = offset[i];
        list[i].adjust = adjust[i];
    }
    // long products first: the blocks take tiles in turn; then the matrices with teams, the largest teams first
    std::stable_sort(list, list + count, [](const OrthoDesc& p, const OrthoDesc& q) {
        if (!p.team != !q.team) return !p.team;
        if (p.team) return p.team > q.team;
        return p.m != q.m ? p.m > q.m : p.n > q.n;
    });
    int64_t general = 0, spans = 0, slots = 0;
    for (; general < count && !list[general].team;) ++general;
    for (int64_t i = 0; i < count; ++i) {
        list[i].span0 = spans;
        spans += or_spans((int64_t)list[i].m * list[i].n);
        list[i].slot0 = slots;
        slots += list[i].team;
    }
    const OrthoShape shape = or_choose(list, general, false);
    const int bn_sym = shape.bn_sym, bn_upd = shape.bn_upd, pair = shape.pair;
    int64_t waves = 0, most = 0, most_items = 0;
    int64_t* wave = plan + 8;
    OrthoDesc at = {};
    for (int64_t i = 0; i < general; ++i) {
        const int m = list[i].m, n = list[i].n;
        const int64_t bytes = or_tiles_bytes(m, n);
        if (i == 0 || at.ws + bytes > ORTHO_BUDGET) {  // the next launch
            if (i) wave += 7;
            at = OrthoDesc{};
            wave[0] = i;
            ++waves;
        }
        list[i].ws = at.ws, list[i].conv0 = at.conv0, list[i].sym0 = at.sym0, list[i].upd0 = at.upd0;
        at.ws += bytes;
        at.conv0 += (int64_t)or_mb(m) * or_b64(n);
        at.sym0 += or_syms(m, bn_sym, pair, shape.mirror);
        at.upd0 += or_upds(m, n, bn_upd, pair);
        const int split = or_split_of(m, n, shape);
        const int64_t items = split * or_syms(m, bn_sym, pair, shape.mirror);
        list[i].split = split, list[i].gram0 = at.gram0, list[i].part0 = at.part0;
        at.gram0 += items;
        if (split > 1) at.part0 += items;
        if (at.part0 > most_items) most_items = at.part0;
        if (at.ws > most) most = at.ws;
        wave[1] = i + 1 - wave[0], wave[2] = at.conv0, wave[3] = at.sym0, wave[4] = at.upd0;
        wave[5] = at.gram0, wave[6] = at.part0;
    }
    plan[0] = or_up(256 + or_arrived_bytes(most_items)) + or_up(spans * 8) + or_up(or_parts_bytes(most_items, shape)) + most;
    plan[1] = spans, plan[2] = waves, plan[3] = bn_sym, plan[4] = bn_upd;
    plan[5] = pair + 2 * shape.mirror, plan[6] = general, plan[7] = slots;
    plan[8 + 7 * waves] = slots ? list[general].team : 0;  // the clusters' size
    plan[9 + 7 * waves] = most_items;
    return 0;
}

int pbg_muon_step(int64_t count, const void* descriptors, const int64_t* plan, float* grad, float* momentum, float* master,
                  const float* controls, int32_t nesterov, int32_t steps, float a, float b, float c, double eps,
                  void* workspace, int64_t workspace_bytes, uint32_t* skipped, uint32_t* error, void* stream) {
    PBG_REQUIRE(count >= 1 && descriptors && plan && grad && momentum && master && controls && workspace && skipped && error,
                "muon_step: null argument");
    PBG_REQUIRE(eps >= 0.0, "muon_step: epsilon must not be negative");
    PBG_REQUIRE((uintptr_t)workspace % 256 == 0 && workspace_bytes >= plan[0], "muon_step: workspace too small or unaligned");
    int rc = or_check_polynomial(steps, a, b, c);
    if (rc) return rc;
    cudaStream_t s = as_stream(stream);
    unsigned char* w = static_cast<unsigned char*>(workspace);
    OrthoArgs O = {};
    const int64_t waves = plan[2], most_items = plan[9 + 7 * waves];
    const OrthoShape shape = {(int)plan[3], (int)plan[4], (int)plan[5] & 1, (int)plan[5] >> 1, 0.0};
    O.barrier = reinterpret_cast<uint32_t*>(w);
    O.arrived = reinterpret_cast<uint32_t*>(w + 256);
    w += or_up(256 + or_arrived_bytes(most_items));
    O.sums = reinterpret_cast<double*>(w);
    w += or_up(plan[1] * 8);
    O.parts = reinterpret_cast<float*>(w);
    O.tiles = w + or_up(or_parts_bytes(most_items, shape));
    O.bn_sym = (int)plan[3], O.bn_upd = (int)plan[4], O.pair = (int)plan[5] & 1, O.mirror = (int)plan[5] >> 1;
    O.steps = steps, O.a = a, O.b = b, O.c = c, O.eps = eps;
    O.grad = grad, O.momentum = momentum, O.master = master, O.controls = controls;
    O.nesterov = nesterov, O.bad = skipped, O.error = error;
    O.aligned = (uintptr_t)grad % 16 == 0 && (uintptr_t)momentum % 16 == 0 && (uintptr_t)master % 16 == 0;
    rc = cuda_status(cudaMemsetAsync(skipped, 0, 4, s), "muon_step: status");
    if (rc) return rc;
    const OrthoDesc* list = static_cast<const OrthoDesc*>(descriptors);
    O.list = list, O.count = count, O.spans = plan[1];
    rc = or_squares(O, s);  // of all matrices: every direction is checked before anything is written
    if (rc) return rc;
    for (int64_t i = 0; i < waves; ++i) {
        const int64_t* wave = plan + 8 + 7 * i;
        O.list = list + wave[0], O.count = wave[1];
        O.convs = wave[2], O.syms = wave[3], O.upds = wave[4], O.grams = wave[5];
        rc = or_products(O, or_arrived_bytes(wave[6]), s);
        if (rc) return rc;
    }
    if (plan[7]) {
        const int64_t general = plan[6];
        O.list = list + general, O.count = count - general, O.slots = plan[7];
        return or_teams(O, (int)plan[8 + 7 * waves], s);
    }
    return 0;
}

}  // extern "C"
