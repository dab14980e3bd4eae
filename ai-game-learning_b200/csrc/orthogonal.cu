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
// on and above the diagonal are computed, the others mirrored), X' = B X, run on the tensor cores
// (tcgen05, fp32 accumulation in tensor memory) over all matrices of the call at once, a persistent CTA
// per SM.
//
// Precision.  16-bit operands alone are not enough: an error in X in the direction of a small singular
// value grows by a = 3.4 each step, so X is carried as a pair of fp16 numbers hi + lo of 2^14 X (22
// significant bits; every |x| <= sigma_max <= 2 keeps hi in range).  With fp32 output, and in the
// optimizer's transition, A and B are pairs too (2^13 A, 2^12 B) and each product takes three passes,
// hi hi + hi lo + lo hi, leaving errors of about 2^-22: at or below what fp32 operands give.  With bf16
// output of matrices whose short side is at least ORTHO_SINGLE the symmetric matrices are single fp16
// numbers (error 2^-12 that does not grow: about 8e-4 of the result's norm, where bf16 rounding alone is
// 1.7e-3): one pass for A and B, two for X'.  The tensor cores truncate as they accumulate, a bias that
// grows with the length of the sum, so a sum is taken from tensor memory every ORTHO_CHUNK * 64 terms
// and added up in fp32 registers.
//
// Layout.  X, A and B live in the workspace as 128 x 64 tiles of 16 KB, hi then lo, already in the
// 128-byte-swizzled form that the tensor cores read from shared memory, so operands of any matrix of any
// size are fetched by plain contiguous bulk copies (no tensor maps), and one tile serves both as a
// K-major operand (X X^T) and, by halves, as an MN-major one (B X).  Short sides are padded with zeros to
// 128 and long sides to 64.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "pbg_common.cuh"

namespace pbg {

constexpr int ORTHO_CHUNK = 4;         // k-blocks of 64 summed in tensor memory
constexpr int ORTHO_EPI_WARPS = 16;
constexpr int ORTHO_THREADS = 64 + 32 * ORTHO_EPI_WARPS;
constexpr int ORTHO_RING = 192 * 1024;  // operand stages
constexpr int ORTHO_STAGES = 8;         // at most
constexpr int ORTHO_BLOCK = 2048;       // an epilogue warp's staging block
constexpr int ORTHO_SMEM = 1024 + ORTHO_RING + ORTHO_EPI_WARPS * ORTHO_BLOCK;
constexpr int ORTHO_SPAN = ORTHO_THREADS * 16;  // elements whose squares one block sums
constexpr int ORTHO_TILE = 32768;       // bytes of a 128 x 64 tile, hi and lo
constexpr uint32_t ORTHO_WAIT_TRIES = 1u << 24;
constexpr float ORTHO_SX = 16384.0f, ORTHO_SA = 8192.0f, ORTHO_SB = 4096.0f;

struct OrthoDesc {
    int64_t src;     // first element
    int64_t ws;      // bytes of workspace before this matrix's tiles: X, X', A, B
    int64_t span0;   // spans, conversion tiles, symmetric and update tiles of the matrices before it
    int64_t conv0, sym0, upd0;
    int32_t m, n;    // short and long side
    int32_t tall;    // stored n x m
    float adjust;
};

struct OrthoArgs {
    const OrthoDesc* list;  // device, or null: `count` matrices like `one`, `one`'s sizes apart
    OrthoDesc one;
    int64_t one_src, one_ws, one_span, one_conv, one_sym, one_upd;
    int64_t count, spans, convs, syms, upds;  // totals
    int bn_sym, bn_upd;  // output tile widths
    int steps, precise;  // precise: A and B as pairs
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
    uint32_t* barrier;
    uint32_t* error;
    int phase0, phase1;
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
// columns of 8 k-rows an atom, the next k-rows 1024 bytes on, the next 64 columns `lbo` bytes on)
__device__ __forceinline__ uint64_t or_desc(uint32_t addr, uint32_t lbo) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}
// kind::f16: fp16 x fp16 -> fp32, M 128, A K-major, B K-major or MN-major
__device__ __forceinline__ uint32_t or_idesc(int n, int mn_major) {
    return (1u << 4) | ((uint32_t)mn_major << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void or_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void or_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void or_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void or_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void or_tmem_add32(uint32_t taddr, float* acc) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int j = 0; j < 32; ++j) acc[j] += __uint_as_float(r[j]);
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
__host__ __device__ __forceinline__ int64_t or_x_bytes(int m, int n) { return (int64_t)or_mb(m) * or_b64(n) * ORTHO_TILE; }
__host__ __device__ __forceinline__ int64_t or_a_bytes(int m) { return (int64_t)or_mb(m) * 2 * or_mb(m) * ORTHO_TILE; }
// symmetric tiles of row block i: from column 128 i on
__host__ __device__ __forceinline__ int or_sym_row(int m, int i, int bn) { return (or_b64(m) * 64 - i * 128 + bn - 1) / bn; }

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

struct OrthoShared {
    uint64_t full[ORTHO_STAGES], empty[ORTHO_STAGES], acc_full[2], acc_empty[2], done;
    double reduce[ORTHO_THREADS / 32];
    double norm;
    int64_t norm_of;
    uint32_t tmem;
    int ok;
    volatile int abort_flag;
};

__device__ __forceinline__ double or_block_sum(double v, OrthoShared& S) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) S.reduce[threadIdx.x >> 5] = v;
    __syncthreads();
    double sum = 0.0;
    for (int w = 0; w < ORTHO_THREADS / 32; ++w) sum += S.reduce[w];
    return sum;
}

// squares of each matrix's direction, a sum per span (fp64: no overflow or underflow at any fp32 scale)
__device__ void or_phase_squares(const OrthoArgs& O, OrthoShared& S) {
    const OrthoDirection k = or_controls(O);
    for (int64_t t = blockIdx.x; t < O.spans; t += gridDim.x) {
        const OrthoDesc d = or_get(O, or_find(O, t, &OrthoDesc::span0, O.one_span));
        const int64_t total = (int64_t)d.m * d.n;
        const int64_t begin = (t - d.span0) * ORTHO_SPAN;
        const int64_t end = begin + ORTHO_SPAN < total ? begin + ORTHO_SPAN : total;
        double sum = 0.0;
        bool bad = false;
        for (int64_t i = begin + threadIdx.x; i < end; i += ORTHO_THREADS) {
            float u;
            if (O.x) {
                u = or_load(O.x, O.x_type, d.src + i);
            } else {
                const float g = O.grad[d.src + i];
                u = or_direction(k, g, or_momentum(k, g, O.momentum[d.src + i]));
                bad |= !isfinite(u);
            }
            sum += (double)u * (double)u;
        }
        if (bad) atomicExch(O.bad, 1u);
        sum = or_block_sum(sum, S);
        if (threadIdx.x == 0) O.sums[t] = sum;
    }
}

__device__ __forceinline__ void or_split(float v, __half& hi, __half& lo) {
    hi = __float2half_rn(v);
    lo = __float2half_rn(v - __half2float(hi));
}

// the normalised direction as tiles of pairs (and the momentum, where there is one)
__device__ void or_phase_convert(const OrthoArgs& O, OrthoShared& S) {
    const OrthoDirection k = or_controls(O);
    if (threadIdx.x == 0) S.norm_of = -1;
    __syncthreads();
    for (int64_t t = blockIdx.x; t < O.convs; t += gridDim.x) {
        const int64_t which = or_find(O, t, &OrthoDesc::conv0, O.one_conv);
        const OrthoDesc d = or_get(O, which);
        const int64_t total = (int64_t)d.m * d.n;
        if (S.norm_of != which) {
            const int64_t spans = (total + ORTHO_SPAN - 1) / ORTHO_SPAN;
            double sum = 0.0;
            for (int64_t i = threadIdx.x; i < spans; i += ORTHO_THREADS) sum += __ldcg(O.sums + d.span0 + i);
            sum = or_block_sum(sum, S);
            __syncthreads();
            if (threadIdx.x == 0) {
                S.norm = sqrt(sum);
                S.norm_of = which;
            }
            __syncthreads();
        }
        const float scale = (float)((double)ORTHO_SX / (S.norm + O.eps));
        // a scale beyond fp32 belongs to a direction of (sub)normal smallness: taken in fp64 then
        const bool plain = scale < 1.0e30f;
        const double wide = (double)ORTHO_SX / (S.norm + O.eps);
        const int nb = or_b64(d.n);
        const int local = (int)(t - d.conv0);
        const int row0 = (local / nb) * 128, col0 = (local % nb) * 64;
        unsigned char* tile = O.tiles + d.ws + (int64_t)local * ORTHO_TILE;
        for (int q = threadIdx.x; q < 1024; q += ORTHO_THREADS) {
            const int r = q >> 3, chunk = q & 7;
            const int row = row0 + r, col = col0 + chunk * 8;
            __align__(16) __half hi[8];
            __align__(16) __half lo[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float u = 0.0f;
                if (row < d.m && col + e < d.n) {
                    const int64_t i = d.src + (d.tall ? (int64_t)(col + e) * d.m + row : (int64_t)row * d.n + col + e);
                    if (O.x) {
                        u = or_load(O.x, O.x_type, i);
                    } else {
                        const float g = O.grad[i];
                        const float m = or_momentum(k, g, O.momentum[i]);
                        O.momentum[i] = m;
                        u = or_direction(k, g, m);
                    }
                    u = plain ? u * scale : (float)((double)u * wide);
                }
                or_split(u, hi[e], lo[e]);
            }
            const int at = r * 128 + ((chunk ^ (r & 7)) << 4);
            *reinterpret_cast<uint4*>(tile + at) = *reinterpret_cast<uint4*>(hi);
            *reinterpret_cast<uint4*>(tile + 16384 + at) = *reinterpret_cast<uint4*>(lo);
        }
    }
}

// ------------------------------------------------------------ products

enum { OR_GRAM = 0, OR_SQUARE = 1, OR_UPDATE = 2 };

// one output tile: row block, first column, width, and where its operands lie
struct OrthoTile {
    OrthoDesc d;
    int i, c0, width, kblocks;
    const unsigned char* a;  // tiles of the row operand: k-block kb at a + kb * ORTHO_TILE
    const unsigned char* b;  // the other operand's tiles
    int64_t b_row;           // bytes between its row blocks
    unsigned char *x_next, *amat, *bmat;
};

__device__ __forceinline__ OrthoTile or_tile(const OrthoArgs& O, int kind, int step, int64_t t) {
    OrthoTile T;
    const bool sym = kind != OR_UPDATE;
    T.d = or_get(O, sym ? or_find(O, t, &OrthoDesc::sym0, O.one_sym) : or_find(O, t, &OrthoDesc::upd0, O.one_upd));
    const int m64 = or_b64(T.d.m), nb = or_b64(T.d.n), mb = or_mb(T.d.m);
    const int64_t xb = or_x_bytes(T.d.m, T.d.n), ab = or_a_bytes(T.d.m);
    unsigned char* base = O.tiles + T.d.ws;
    unsigned char* x = base + (step & 1 ? xb : 0);
    T.x_next = base + (step & 1 ? 0 : xb);
    T.amat = base + 2 * xb;
    T.bmat = T.amat + ab;
    int local = (int)(t - (sym ? T.d.sym0 : T.d.upd0));
    if (sym) {
        T.i = 0;
        for (int n; local >= (n = or_sym_row(T.d.m, T.i, O.bn_sym)); ++T.i) local -= n;
        T.c0 = T.i * 128 + local * O.bn_sym;
        T.width = min(O.bn_sym, m64 * 64 - T.c0);
    } else {
        const int across = (nb * 64 + O.bn_upd - 1) / O.bn_upd;
        T.i = local / across;
        T.c0 = (local % across) * O.bn_upd;
        T.width = min(O.bn_upd, nb * 64 - T.c0);
    }
    if (kind == OR_GRAM) {
        T.kblocks = nb;
        T.b_row = (int64_t)nb * ORTHO_TILE;
        T.a = x + T.i * T.b_row;
        T.b = x;
    } else if (kind == OR_SQUARE) {
        T.kblocks = m64;
        T.b_row = (int64_t)2 * mb * ORTHO_TILE;
        T.a = T.amat + T.i * T.b_row;
        T.b = T.amat;
    } else {
        T.kblocks = m64;
        T.b_row = (int64_t)nb * ORTHO_TILE;
        T.a = T.bmat + (int64_t)T.i * 2 * mb * ORTHO_TILE;
        T.b = x;
    }
    return T;
}

// A thread's 64 finished values of one row as a 128 x 64 tile's row, hi or lo, by way of the warp's staging
// block, 16 rows at a time (rows of 128 bytes are contiguous in the tile, so each half is one bulk copy).
__device__ __forceinline__ void or_store_rows(uint32_t blk, unsigned char* dst, int lane, const float* v, bool low) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncwarp();
        if ((lane >> 4) == half) {
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float x0 = v[8 * q + 2 * j], x1 = v[8 * q + 2 * j + 1];
                    __half2 h = __floats2half2_rn(x0, x1);
                    if (low) {
                        const float2 f = __half22float2(h);
                        h = __floats2half2_rn(x0 - f.x, x1 - f.y);
                    }
                    w[j] = *reinterpret_cast<uint32_t*>(&h);
                }
                const uint32_t addr = blk + (uint32_t)(lane & 15) * 128u + (uint32_t)((q ^ (lane & 7)) << 4);
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                             "r"(w[3])
                             : "memory");
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
            asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst + half * 2048), "r"(blk),
                         "r"(2048u)
                         : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
    }
}

__device__ __forceinline__ void or_write_out(const OrthoArgs& O, const OrthoDesc& d, float lr, float shrink, int64_t i,
                                             float v) {
    if (!O.x) {
        O.master[i] = O.master[i] * shrink - lr * d.adjust * v;
    } else if (O.out_type == 0) {
        static_cast<float*>(O.out)[i] = v;
    } else if (O.out_type == 1) {
        static_cast<__nv_bfloat16*>(O.out)[i] = __float2bfloat16_rn(v);
    } else {
        static_cast<__half*>(O.out)[i] = __float2half_rn(v);
    }
}

// what an epilogue warp does with its 32 rows x 64 columns (rows row0 + lane, column block cb of 64)
__device__ __forceinline__ void or_finish(const OrthoArgs& O, int kind, bool last, const OrthoTile& T, int row, int cb,
                                          uint32_t blk, int lane, float* v) {
    const int m64 = or_b64(T.d.m), mb = or_mb(T.d.m), nb = or_b64(T.d.n);
    const int r0 = row - lane;  // multiple of 32
    if (kind != OR_UPDATE) {
        unsigned char* dst = kind == OR_GRAM ? T.amat : T.bmat;
        const int64_t row_bytes = (int64_t)2 * mb * ORTHO_TILE;
        const bool mirror = cb * 64 >= (T.i + 1) * 128;
        // the mirrored place of (row, cb * 64 + j): tile row block cb / 2, column block row / 64
        const int64_t mirror0 = (int64_t)(cb >> 1) * row_bytes + (int64_t)(row >> 6) * ORTHO_TILE;
        const int mc = row & 63;
        if (kind == OR_GRAM) {
#pragma unroll
            for (int j = 0; j < 64; ++j) v[j] *= ORTHO_SA / (ORTHO_SX * ORTHO_SX);
        } else {
            const float fa = O.a * ORTHO_SB, fb = O.b * (ORTHO_SB / ORTHO_SA), fc = O.c * (ORTHO_SB / (ORTHO_SA * ORTHO_SA));
            const unsigned char* am = T.amat + mirror0;
#pragma unroll
            for (int j = 0; j < 64; ++j) {
                // A(col, row) = A(row, col): lanes read along a row
                const int mr = (cb & 1) * 64 + j;
                const int at = mr * 128 + (((mc >> 3) ^ (mr & 7)) << 4) + (mc & 7) * 2;
                float x = 0.0f;  // rows past the last 64-row block are nobody's operand
                if (row < m64 * 64) x = __half2float(__ushort_as_half(__ldcg(reinterpret_cast<const unsigned short*>(am + at))));
                if (O.precise && row < m64 * 64)
                    x += __half2float(__ushort_as_half(__ldcg(reinterpret_cast<const unsigned short*>(am + 16384 + at))));
                v[j] = fmaf(fc, v[j], fb * x) + (row == cb * 64 + j ? fa : 0.0f);
            }
        }
        unsigned char* tile = dst + T.i * row_bytes + (int64_t)cb * ORTHO_TILE + (r0 & 127) * 128;
        or_store_rows(blk, tile, lane, v, false);
        if (O.precise) or_store_rows(blk, tile + 16384, lane, v, true);
        if (mirror) {
            unsigned char* mt = dst + mirror0;
#pragma unroll
            for (int j = 0; j < 64; ++j) {
                const int mr = (cb & 1) * 64 + j;
                const int at = mr * 128 + (((mc >> 3) ^ (mr & 7)) << 4) + (mc & 7) * 2;
                __half hi, lo;
                or_split(v[j], hi, lo);
                *reinterpret_cast<__half*>(mt + at) = hi;
                if (O.precise) *reinterpret_cast<__half*>(mt + 16384 + at) = lo;
            }
        }
    } else if (!last) {
#pragma unroll
        for (int j = 0; j < 64; ++j) v[j] *= 1.0f / ORTHO_SB;
        unsigned char* tile = T.x_next + ((int64_t)T.i * nb + cb) * ORTHO_TILE + (r0 & 127) * 128;
        or_store_rows(blk, tile, lane, v, false);
        or_store_rows(blk, tile + 16384, lane, v, true);
    } else {
        const float lr = O.x ? 0.0f : O.controls[0];
        const float shrink = O.x ? 1.0f : 1.0f - lr * O.controls[2];
        if (T.d.tall) {
            if (row < T.d.m) {
#pragma unroll
                for (int j = 0; j < 64; ++j) {
                    const int col = cb * 64 + j;
                    if (col < T.d.n)
                        or_write_out(O, T.d, lr, shrink, T.d.src + (int64_t)col * T.d.m + row, v[j] * (1.0f / (ORTHO_SB * ORTHO_SX)));
                }
            }
        } else {
            // 32 rows x 16 columns at a time by way of the staging block, so that lanes write along rows
            if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            __syncwarp();
#pragma unroll
            for (int p = 0; p < 4; ++p) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint32_t addr = blk + (uint32_t)lane * 64u + (uint32_t)((q ^ ((lane >> 1) & 3)) << 4);
                    asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v[16 * p + 4 * q]),
                                 "f"(v[16 * p + 4 * q + 1]), "f"(v[16 * p + 4 * q + 2]), "f"(v[16 * p + 4 * q + 3])
                                 : "memory");
                }
                __syncwarp();
#pragma unroll
                for (int it = 0; it < 16; ++it) {
                    const int rr = it * 2 + (lane >> 4), cc = lane & 15;
                    float x;
                    const uint32_t addr =
                        blk + (uint32_t)rr * 64u + (uint32_t)(((cc >> 2) ^ ((rr >> 1) & 3)) << 4) + (uint32_t)(cc & 3) * 4u;
                    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(addr) : "memory");
                    const int col = cb * 64 + p * 16 + cc;
                    if (r0 + rr < T.d.m && col < T.d.n)
                        or_write_out(O, T.d, lr, shrink, T.d.src + (int64_t)(r0 + rr) * T.d.n + col, x * (1.0f / (ORTHO_SB * ORTHO_SX)));
                }
                __syncwarp();
            }
        }
    }
}

struct OrthoPipe {
    uint32_t full, empty;  // parity of each stage's next use, a bit a stage
    uint32_t acc;          // accumulators used
};

__device__ void or_phase_product(const OrthoArgs& O, OrthoShared& S, OrthoPipe& P, uint32_t ring, int kind, int step) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t tiles = kind == OR_UPDATE ? O.upds : O.syms;
    const int bn = kind == OR_UPDATE ? O.bn_upd : O.bn_sym;
    const int pa = O.precise ? 2 : 1, pb = O.precise || kind == OR_UPDATE ? 2 : 1;
    const uint32_t a_bytes = pa * 16384u, b_part = (uint32_t)bn * 128u;
    const uint32_t stage_bytes = a_bytes + pb * b_part;
    const int stages = min(ORTHO_STAGES, (int)(ORTHO_RING / stage_bytes));
    if (warp == 0) {
        if (lane == 0) {
            asm volatile("fence.proxy.async;" ::: "memory");
            bool ok = true;
            int s = 0;
            uint32_t used = 0;
            for (int64_t t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
                const OrthoTile T = or_tile(O, kind, step, t);
                const int pieces = T.width >> 6;
                for (int kb = 0; kb < T.kblocks; ++kb) {
                    if (!or_wait(or_smem(&S.empty[s]), ((P.empty >> s) & 1u) ^ 1u, &S.abort_flag)) {
                        ok = false;
                        break;
                    }
                    P.empty ^= 1u << s;
                    used |= 1u << s;
                    const uint32_t bar = or_smem(&S.full[s]), sa = ring + s * stage_bytes, sb = sa + a_bytes;
                    or_expect_tx(bar, a_bytes + (uint32_t)(pb * pieces) * 8192u);
                    or_bulk_load(sa, T.a + (int64_t)kb * ORTHO_TILE, a_bytes, bar);
                    for (int p = 0; p < pieces; ++p) {
                        // 64 rows of k-block kb (K-major), or 64 k-rows of a column block (MN-major)
                        const int cb = (T.c0 >> 6) + p;
                        const unsigned char* src =
                            kind == OR_UPDATE ? T.b + (kb >> 1) * T.b_row + (int64_t)cb * ORTHO_TILE + (kb & 1) * 8192
                                              : T.b + (cb >> 1) * T.b_row + (int64_t)kb * ORTHO_TILE + (cb & 1) * 8192;
                        or_bulk_load(sb + p * 8192u, src, 8192u, bar);
                        if (pb == 2) or_bulk_load(sb + b_part + p * 8192u, src + 16384, 8192u, bar);
                    }
                    if (++s == stages) s = 0;
                }
            }
            if (!ok) {
                atomicCAS(O.error, 0u, 1u);
                S.abort_flag = 1;
            }
            if (S.abort_flag) {  // every copy under way lands before the block can end
                for (int q = 0; q < stages; ++q)
                    for (uint32_t i = 0; ((used >> q) & 1u) && i < ORTHO_WAIT_TRIES &&
                                         !or_try_wait(or_smem(&S.full[q]), ((P.empty >> q) & 1u) ^ 1u); ++i) {
                    }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            bool ok = true;
            int s = 0;
            const int mn = kind == OR_UPDATE;
            const uint32_t b_step = mn ? 2048u : 32u, lbo = mn ? 8192u : 16u;
            for (int64_t t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
                const OrthoTile T = or_tile(O, kind, step, t);
                const uint32_t idesc = or_idesc(T.width, mn);
                for (int k0 = 0; ok && k0 < T.kblocks; k0 += ORTHO_CHUNK, ++P.acc) {
                    const uint32_t b = P.acc & 1u;
                    if (!or_wait(or_smem(&S.acc_empty[b]), ((P.acc >> 1) & 1u) ^ 1u, &S.abort_flag)) {
                        ok = false;
                        break;
                    }
                    or_fence_after();
                    const uint32_t d = S.tmem + b * 256u;
                    const int k1 = min(k0 + ORTHO_CHUNK, T.kblocks);
                    for (int kb = k0; kb < k1; ++kb) {
                        if (!or_wait(or_smem(&S.full[s]), (P.full >> s) & 1u, &S.abort_flag)) {
                            ok = false;
                            break;
                        }
                        P.full ^= 1u << s;
                        or_fence_after();
                        const uint32_t sa = ring + s * stage_bytes, sb = sa + a_bytes;
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks) {
                            const uint64_t ah = or_desc(sa + ks * 32, 16), bh = or_desc(sb + ks * b_step, lbo);
                            if (pa == 2) or_mma(d, or_desc(sa + 16384 + ks * 32, 16), bh, idesc, kb > k0 || ks > 0);
                            if (pb == 2) or_mma(d, ah, or_desc(sb + b_part + ks * b_step, lbo), idesc, kb > k0 || ks > 0 || pa == 2);
                            or_mma(d, ah, bh, idesc, kb > k0 || ks > 0 || pb == 2);
                        }
                        or_commit(or_smem(&S.empty[s]));
                        if (++s == stages) s = 0;
                    }
                    if (ok) or_commit(or_smem(&S.acc_full[b]));
                }
            }
            if (!ok) {
                atomicCAS(O.error, 0u, 2u);
                S.abort_flag = 1;
            }
        }
    } else {
        const int e = warp - 2, quad = warp & 3, part = e >> 2;
        const uint32_t blk = ring + ORTHO_RING + (uint32_t)e * ORTHO_BLOCK;
        const bool last = kind == OR_UPDATE && step == O.steps - 1;
        bool ok = true;
        for (int64_t t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
            const OrthoTile T = or_tile(O, kind, step, t);
            const bool mine = part < (T.width >> 6);
            float v[64];
#pragma unroll
            for (int j = 0; j < 64; ++j) v[j] = 0.0f;
            for (int k0 = 0; k0 < T.kblocks; k0 += ORTHO_CHUNK, ++P.acc) {
                const uint32_t b = P.acc & 1u;
                ok = __all_sync(0xffffffffu, or_wait(or_smem(&S.acc_full[b]), (P.acc >> 1) & 1u, &S.abort_flag));
                if (!ok) break;
                or_fence_after();
                if (mine) {
                    const uint32_t taddr = S.tmem + ((uint32_t)(quad * 32) << 16) + b * 256u + (uint32_t)(part * 64);
                    or_tmem_add32(taddr, v);
                    or_tmem_add32(taddr + 32, v + 32);
                }
                or_fence_before();
                or_arrive(or_smem(&S.acc_empty[b]));
            }
            if (ok && mine) or_finish(O, kind, last, T, T.i * 128 + quad * 32 + lane, (T.c0 >> 6) + part, blk, lane, v);
        }
        if (!ok) {
            if (lane == 0) atomicCAS(O.error, 0u, 3u);
            S.abort_flag = 1;
        }
        // the staging block's copies have been written before anyone reads them
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        __syncwarp();
    }
    asm volatile("fence.proxy.async;" ::: "memory");
    __syncthreads();
}

// All blocks (launched cooperatively, so all run); bounded.
__device__ bool or_grid_sync(const OrthoArgs& O, OrthoShared& S, uint32_t& target) {
    target += gridDim.x;
    asm volatile("fence.proxy.async;" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        uint32_t seen = atomicAdd(O.barrier, 1u) + 1u;
        for (uint32_t i = 0; (int32_t)(seen - target) < 0 && i < ORTHO_WAIT_TRIES; ++i)
            asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(O.barrier) : "memory");
        const bool ok = (int32_t)(seen - target) >= 0;
        if (!ok) atomicCAS(O.error, 0u, 4u);
        __threadfence();
        S.ok = ok && !S.abort_flag;
    }
    __syncthreads();
    asm volatile("fence.proxy.async;" ::: "memory");
    return S.ok != 0;
}

// the transition where a direction is not finite: the matrices' gradients are cleared
__device__ void or_phase_clear(const OrthoArgs& O) {
    for (int64_t t = blockIdx.x; t < O.convs; t += gridDim.x) {
        const OrthoDesc d = or_get(O, or_find(O, t, &OrthoDesc::conv0, O.one_conv));
        const int64_t total = (int64_t)d.m * d.n;
        const int64_t begin = (t - d.conv0) * 8192;  // a tile's worth of elements in storage order
        const int64_t end = begin + 8192 < total ? begin + 8192 : total;
        for (int64_t i = begin + threadIdx.x; i < end; i += ORTHO_THREADS) O.grad[d.src + i] = 0.0f;
    }
}

// Phases: 0 squares, 1 conversion, then per step the Gram matrix, its polynomial, and the update.
__global__ void __launch_bounds__(ORTHO_THREADS, 1) orthogonalize_kernel(const __grid_constant__ OrthoArgs O) {
    extern __shared__ __align__(16) unsigned char or_raw[];
    __shared__ __align__(8) OrthoShared S;
    const uint32_t ring = (or_smem(or_raw) + 1023u) & ~1023u;
    const int warp = threadIdx.x >> 5;
    const bool products = O.phase1 > 2;
    if (threadIdx.x == 0) {
        S.abort_flag = 0;
        for (int s = 0; s < ORTHO_STAGES; ++s) {
            or_mbar_init(or_smem(&S.full[s]), 1);
            or_mbar_init(or_smem(&S.empty[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            or_mbar_init(or_smem(&S.acc_full[b]), 1);
            or_mbar_init(or_smem(&S.acc_empty[b]), 32 * ORTHO_EPI_WARPS);
        }
        or_mbar_init(or_smem(&S.done), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (products && warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(or_smem(&S.tmem)), "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    or_fence_before();
    __syncthreads();
    or_fence_after();
    OrthoPipe P = {0u, 0u, 0u};
    uint32_t target = 0;
    for (int phase = O.phase0; phase < O.phase1; ++phase) {
        if (phase > O.phase0 && !or_grid_sync(O, S, target)) break;
        const bool bad = phase > 0 && !O.x && __ldcg(O.bad) != 0u;
        if (phase == 0) or_phase_squares(O, S);
        else if (bad) {
            if (phase == 1) or_phase_clear(O);
        } else if (phase == 1) {
            or_phase_convert(O, S);
        } else {
            or_phase_product(O, S, P, ring, (phase - 2) % 3, (phase - 2) / 3);
            if (S.abort_flag) break;
        }
    }
    __syncthreads();
    if (products && warp == 1) {
        if ((threadIdx.x & 31) == 0) {
            // nothing that this thread issued is under way when the memory is freed
            or_commit(or_smem(&S.done));
            for (uint32_t i = 0; i < ORTHO_WAIT_TRIES && !or_try_wait(or_smem(&S.done), 0u); ++i) {
            }
        }
        __syncwarp();
        or_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(S.tmem), "r"(512u) : "memory");
    }
}

// ------------------------------------------------------------ host

constexpr int64_t ORTHO_BUDGET = 1ll << 30;  // bytes of tiles that one launch works in, where a matrix alone does not need more
constexpr int ORTHO_SINGLE = 512;

static int64_t or_tiles_bytes(int m, int n) { return 2 * or_x_bytes(m, n) + 2 * or_a_bytes(m); }
static int64_t or_spans(int64_t total) { return (total + ORTHO_SPAN - 1) / ORTHO_SPAN; }
static int64_t or_syms(int m, int bn) {
    int64_t n = 0;
    for (int i = 0; i < or_mb(m); ++i) n += or_sym_row(m, i, bn);
    return n;
}
static int64_t or_upds(int m, int n, int bn) { return (int64_t)or_mb(m) * ((or_b64(n) * 64 + bn - 1) / bn); }

static OrthoDesc or_make(int64_t rows, int64_t cols) {
    OrthoDesc d = {};
    d.tall = rows > cols;
    d.m = (int)(d.tall ? cols : rows);
    d.n = (int)(d.tall ? rows : cols);
    d.adjust = 1.0f;
    return d;
}

// Output tile width, by an estimate of the busiest SM's cycles: a k-block of 64 costs 12 instructions of
// 48, 64 or 128 cycles at widths 64, 128 and 256 (the narrow ones wait for shared memory), an output tile
// some 1,500 cycles and 6 a column to finish.  Wide tiles carry long products (256: 0.9 of the cycles per
// multiply-add that 128 takes, 0.67 of 64), narrow ones spread a few small matrices over more SMs.
struct OrthoWidths {
    double sum[2][3], top[2][3];
};
static const int OR_WIDTHS[3] = {64, 128, 256};
static void or_weigh(OrthoWidths& W, int m, int n, int64_t count) {
    static const double block[3] = {576.0, 768.0, 1536.0};
    for (int w = 0; w < 3; ++w)
        for (int kind = 0; kind < 2; ++kind) {
            const int bn = OR_WIDTHS[w];
            // the Gram matrix (kind 0) is the longer of the two symmetric products
            const double cost = (kind == 0 ? or_b64(n) : or_b64(m)) * block[w] + 1500.0 + 6.0 * bn;
            W.sum[kind][w] += cost * (double)count * (double)(kind == 0 ? or_syms(m, bn) : or_upds(m, n, bn));
            if (cost > W.top[kind][w]) W.top[kind][w] = cost;
        }
}
static int or_width(const OrthoWidths& W, int kind) {
    int best = 0;
    double least = 0.0;
    for (int w = 0; w < 3; ++w) {
        const double cost = W.sum[kind][w] / sm_count() + W.top[kind][w];
        if (w == 0 || cost < least) best = w, least = cost;
    }
    return OR_WIDTHS[best];
}

static int64_t or_up(int64_t v) { return (v + 1023) / 1024 * 1024; }

static int or_launch(const OrthoArgs& O, cudaStream_t s) {
    static int configured[64] = {0};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        const int rc = cuda_status(cudaFuncSetAttribute(orthogonalize_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, ORTHO_SMEM),
                                   "orthogonalize: shared memory size");
        if (rc) return rc;
        if (dev >= 0 && dev < 64) configured[dev] = 1;
    }
    int64_t want = O.phase0 == 0 ? O.spans : 1;
    if (O.phase1 > 1 && O.convs > want) want = O.convs;
    if (O.phase1 > 2 && O.syms > want) want = O.syms;
    if (O.phase1 > 2 && O.upds > want) want = O.upds;
    const int grid = (int)(want < sm_count() ? want : sm_count());
    int rc = cuda_status(cudaMemsetAsync(O.barrier, 0, 4, s), "orthogonalize: barrier");
    if (rc) return rc;
    void* args[] = {const_cast<OrthoArgs*>(&O)};
    return cuda_status(cudaLaunchCooperativeKernel((const void*)orthogonalize_kernel, dim3((unsigned)grid), dim3(ORTHO_THREADS),
                                                   args, (size_t)ORTHO_SMEM, s),
                       "orthogonalize: cooperative launch");
}

// The fp16 scales hold while no singular value passes 2 and |a + b s^2 + c s^4| stays below 15: followed
// step by step from [0, 1] over a fine grid (the polynomials in use stay within 1.3 and 3.5).
static int or_check_polynomial(int steps, float a, float b, float c) {
    PBG_REQUIRE(steps >= 1 && steps <= 100, "orthogonalize: steps must be in [1,100]");
    double top = 1.0;
    for (int k = 0; k < steps; ++k) {
        double next = 0.0;
        for (int i = 0; i <= 1000; ++i) {
            const double s = top * i / 1000.0, g = s * s, q = a + g * (b + g * c);
            PBG_REQUIRE(q > -15.0 && q < 15.0 && b * g + a < 15.0, "orthogonalize: the coefficients leave the range of the products");
            const double v = s * (q < 0 ? -q : q);
            if (v > next) next = v;
        }
        PBG_REQUIRE(next < 1.9, "orthogonalize: the coefficients let singular values grow past 2");
        const bool same = next <= top;
        top = next > 1.0 ? next : 1.0;
        if (same && k > 0) break;
    }
    return 0;
}

static int64_t or_at_once(int64_t batch, int m, int n) {
    int64_t k = ORTHO_BUDGET / or_tiles_bytes(m, n);
    k = k < 1 ? 1 : k;
    return k < batch ? k : batch;
}

}  // namespace pbg

using namespace pbg;

extern "C" {

int64_t pbg_orthogonalize_workspace(int64_t batch, int64_t rows, int64_t cols) {
    if (batch <= 0 || rows <= 0 || cols <= 0 || rows > 65536 || cols > 65536) return 0;
    const OrthoDesc d = or_make(rows, cols);
    const int64_t k = or_at_once(batch, d.m, d.n);
    return 1024 + or_up(k * or_spans(rows * cols) * 8) + k * or_tiles_bytes(d.m, d.n);
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
    PBG_REQUIRE(workspace_bytes >= pbg_orthogonalize_workspace(batch, rows, cols), "orthogonalize: workspace too small");
    OrthoArgs O = {};
    O.one = or_make(rows, cols);
    const int m = O.one.m, n = O.one.n;
    const int64_t k = or_at_once(batch, m, n);
    unsigned char* w = static_cast<unsigned char*>(workspace);
    O.barrier = reinterpret_cast<uint32_t*>(w);
    O.sums = reinterpret_cast<double*>(w + 1024);
    O.tiles = w + 1024 + or_up(k * or_spans(rows * cols) * 8);
    O.one_src = rows * cols;
    O.one_ws = or_tiles_bytes(m, n);
    O.one_span = or_spans(rows * cols);
    O.one_conv = (int64_t)or_mb(m) * or_b64(n);
    O.steps = steps, O.a = a, O.b = b, O.c = c, O.eps = eps;
    O.x_type = x_type, O.out_type = out_type, O.error = error;
    O.precise = !(out_type == 1 && m >= ORTHO_SINGLE);
    O.phase0 = 0, O.phase1 = 2 + 3 * steps;
    const int64_t xs = x_type == 0 ? 4 : 2, os = out_type == 0 ? 4 : 2;
    for (int64_t at = 0; at < batch; at += k) {
        O.count = batch - at < k ? batch - at : k;
        OrthoWidths W = {};
        or_weigh(W, m, n, O.count);
        O.bn_sym = or_width(W, 0), O.bn_upd = or_width(W, 1);
        O.one_sym = or_syms(m, O.bn_sym), O.one_upd = or_upds(m, n, O.bn_upd);
        O.spans = O.count * O.one_span, O.convs = O.count * O.one_conv;
        O.syms = O.count * O.one_sym, O.upds = O.count * O.one_upd;
        O.x = static_cast<const unsigned char*>(x) + at * rows * cols * xs;
        O.out = static_cast<unsigned char*>(out) + at * rows * cols * os;
        rc = or_launch(O, as_stream(stream));
        if (rc) return rc;
    }
    return 0;
}

int64_t pbg_muon_descriptor_bytes(void) { return (int64_t)sizeof(OrthoDesc); }

int64_t pbg_muon_plan_words(int64_t count) { return count < 0 ? 0 : 8 + 5 * count; }

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
    // long products first: the blocks take tiles in turn
    std::stable_sort(list, list + count, [](const OrthoDesc& p, const OrthoDesc& q) {
        return p.m != q.m ? p.m > q.m : p.n > q.n;
    });
    OrthoWidths W = {};
    for (int64_t i = 0; i < count; ++i) or_weigh(W, list[i].m, list[i].n, 1);
    const int bn_sym = or_width(W, 0), bn_upd = or_width(W, 1);
    int64_t spans = 0, waves = 0, most = 0;
    int64_t* wave = plan + 8;
    OrthoDesc at = {};
    for (int64_t i = 0; i < count; ++i) {
        const int m = list[i].m, n = list[i].n;
        const int64_t bytes = or_tiles_bytes(m, n);
        if (i == 0 || at.ws + bytes > ORTHO_BUDGET) {  // the next launch
            if (i) wave += 5;
            at = OrthoDesc{};
            wave[0] = i;
            ++waves;
        }
        list[i].ws = at.ws, list[i].conv0 = at.conv0, list[i].sym0 = at.sym0, list[i].upd0 = at.upd0;
        list[i].span0 = spans;
        spans += or_spans((int64_t)m * n);
        at.ws += bytes;
        at.conv0 += (int64_t)or_mb(m) * or_b64(n);
        at.sym0 += or_syms(m, bn_sym);
        at.upd0 += or_upds(m, n, bn_upd);
        if (at.ws > most) most = at.ws;
        wave[1] = i + 1 - wave[0], wave[2] = at.conv0, wave[3] = at.sym0, wave[4] = at.upd0;
    }
    plan[0] = 1024 + or_up(spans * 8) + most;
    plan[1] = spans, plan[2] = waves, plan[3] = bn_sym, plan[4] = bn_upd;
    plan[5] = plan[6] = plan[7] = 0;
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
    O.barrier = reinterpret_cast<uint32_t*>(w);
    O.sums = reinterpret_cast<double*>(w + 1024);
    O.tiles = w + 1024 + or_up(plan[1] * 8);
    O.bn_sym = (int)plan[3], O.bn_upd = (int)plan[4];
    O.steps = steps, O.a = a, O.b = b, O.c = c, O.eps = eps;
    O.precise = 1;
    O.grad = grad, O.momentum = momentum, O.master = master, O.controls = controls;
    O.nesterov = nesterov, O.bad = skipped, O.error = error;
    rc = cuda_status(cudaMemsetAsync(skipped, 0, 4, s), "muon_step: status");
    if (rc) return rc;
    const OrthoDesc* list = static_cast<const OrthoDesc*>(descriptors);
    const int64_t waves = plan[2];
    if (waves > 1) {  // every direction is checked before anything is written
        O.list = list, O.count = count, O.spans = plan[1];
        O.phase0 = 0, O.phase1 = 1;
        rc = or_launch(O, s);
        if (rc) return rc;
    }
    for (int64_t i = 0; i < waves; ++i) {
        const int64_t* wave = plan + 8 + 5 * i;
        O.list = list + wave[0], O.count = wave[1];
        O.convs = wave[2], O.syms = wave[3], O.upds = wave[4];
        O.phase0 = waves > 1 ? 1 : 0, O.phase1 = 2 + 3 * steps;
        O.spans = plan[1];
        rc = or_launch(O, s);
        if (rc) return rc;
    }
    return 0;
}

}  // extern "C"
