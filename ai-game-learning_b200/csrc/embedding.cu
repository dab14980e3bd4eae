// Embedding rows by index, times a scale, and the gradient of that lookup.
//
//   forward   out[t, :] = scale * table[index[t], :]
//   backward  dtable[v, :] (+)= scale * sum over t with index[t] == v of grad[t, :]
//
// Both are bound by HBM: the forward reads each looked-up row and writes each output row once, the
// backward reads each incoming row once and writes each table row once.
//
// The backward has no floating-point atomics, so the result is the same in every run on the same data, strides
// and alignment (which decide the vector width, and with it the order of the sums) and the same device.  By size
// (times of the device at 1965 MHz; a call takes 13 to 17 us at least, most of it on the host):
//   - few tokens (EMB_SCAN): no sort.  A warp (up to 256 tokens) or a block per table row looks through all
//     indices, 32 at a time, and adds the rows that match.  512 tokens into 169 x 32: 2.7 us (sorted 15.5).
//   - few table rows (EMB_TABLE): every warp keeps the whole table's sums for its columns in shared memory
//     and adds its share of the tokens' rows in order; then the warps' and the blocks' tables are added in
//     order.  81,920 x 128 fp32 into 13 rows: 15.3 us (sorted 37); 1,000,003 x 128 bf16 into 4 rows: 94 us (125).
//   - small tables of narrow rows (emb_narrow_plan): ranges of rows x 16 columns in a block's shared memory.
//   - else sorted tokens, one cooperative kernel:
//     1. a stable radix sort of (index, position) pairs: least significant digit first, at most 9 bits a
//        pass (the least number of passes, bits shared evenly).  Each sorting block owns a contiguous range
//        of tokens; a pass is its digit histogram, a scan of every digit's counts over the blocks, and the
//        scatter, where a warp ranks 32 keys at a time by matching equal digits.  The blocks that do not
//        sort zero the table meanwhile.
//     2. segment sums over equal shares of the sorted list (not of the table: a row looked up by half of the
//        tokens is shared by as many workers as its tokens deserve).  A worker is a group of 8, 16 or 32
//        lanes with 16-byte vectors side by side on a row; it keeps one fp32 sum per column in registers,
//        four or eight rows in flight.  Runs inside a share are written at once; a run that crosses a border
//        leaves its part in the workspace.
//     3. the parts of each crossing run, added in order.
// An index outside [0, rows) yields a row of zeros, takes no gradient and sets the sticky error word;
// tokens with the padding index take no gradient.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "pbg_common.cuh"

namespace pbg {

enum { EMB_F32 = 0, EMB_BF16 = 1, EMB_F16 = 2 };
constexpr uint32_t EMB_BAD_INDEX = 1, EMB_GAVE_UP = 2;  // bits of the error word
constexpr int EMB_THREADS = 512;
constexpr int EMB_WARPS = EMB_THREADS / 32;
constexpr int EMB_BINS = 512;        // 9-bit digits
constexpr int EMB_MAX_KPT = 8;       // keys a thread ranks per tile
constexpr int EMB_MIN_SHARE = 16;    // sorted tokens a worker takes at least
constexpr int EMB_SERIAL_PARTS = 16; // parts of a run that one worker adds
constexpr uint32_t EMB_WAIT_TRIES = 1u << 24;

template <typename T>
__device__ __forceinline__ float emb_float(T v) {
    if constexpr (std::is_same<T, float>::value) return v;
    else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __bfloat162float(v);
    else return __half2float(v);
}

template <typename T>
__device__ __forceinline__ T emb_zero() {
    if constexpr (std::is_same<T, float>::value) return 0.0f;
    else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __ushort_as_bfloat16(0);
    else return __ushort_as_half(0);
}

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC > 16 ? 16 : sizeof(T) * VEC) EmbVec {
    T v[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ void emb_load(const T* p, float* f) {
    const EmbVec<T, VEC> x = *reinterpret_cast<const EmbVec<T, VEC>*>(p);
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = emb_float(x.v[i]);
}

// VEC values rounded once to the output's type and stored; `type` is uniform over the launch.
template <int VEC>
__device__ __forceinline__ void emb_store(void* base, int64_t at, int type, const float* f) {
    if (type == EMB_F32) {
        constexpr int W = VEC > 4 ? 4 : VEC;
#pragma unroll
        for (int q = 0; q < VEC / W; ++q) {
            EmbVec<float, W> x;
#pragma unroll
            for (int i = 0; i < W; ++i) x.v[i] = f[q * W + i];
            reinterpret_cast<EmbVec<float, W>*>(static_cast<float*>(base) + at)[q] = x;
        }
    } else if (type == EMB_BF16) {
        EmbVec<__nv_bfloat16, VEC> x;
#pragma unroll
        for (int i = 0; i < VEC; ++i) x.v[i] = __float2bfloat16_rn(f[i]);
        *reinterpret_cast<EmbVec<__nv_bfloat16, VEC>*>(static_cast<__nv_bfloat16*>(base) + at) = x;
    } else {
        EmbVec<__half, VEC> x;
#pragma unroll
        for (int i = 0; i < VEC; ++i) x.v[i] = __float2half_rn(f[i]);
        *reinterpret_cast<EmbVec<__half, VEC>*>(static_cast<__half*>(base) + at) = x;
    }
}

template <int VEC>
__device__ __forceinline__ void emb_load_typed(const void* base, int64_t at, int type, float* f) {
    if (type == EMB_F32) {
        constexpr int W = VEC > 4 ? 4 : VEC;
#pragma unroll
        for (int q = 0; q < VEC / W; ++q) emb_load<float, W>(static_cast<const float*>(base) + at + q * W, f + q * W);
    } else if (type == EMB_BF16) {
        emb_load<__nv_bfloat16, VEC>(static_cast<const __nv_bfloat16*>(base) + at, f);
    } else {
        emb_load<__half, VEC>(static_cast<const __half*>(base) + at, f);
    }
}

__device__ __forceinline__ int64_t emb_index(const void* index, int wide, int64_t t) {
    return wide ? __ldg(static_cast<const long long*>(index) + t) : (int64_t)__ldg(static_cast<const int*>(index) + t);
}

// an index outside the table: its bit is set once, so that many such indices do not queue up at one word
__device__ __forceinline__ void emb_bad_index(uint32_t* error) {
    if (!(*reinterpret_cast<volatile uint32_t*>(error) & EMB_BAD_INDEX)) atomicOr(error, EMB_BAD_INDEX);
}

// ---------------------------------------------------------------- forward

struct EmbArgs {
    int64_t tokens, rows, width, ldt;
    const void* index;
    int index64;
    const void* table;
    void* out;
    int out_type;
    int log_lanes;  // lanes side by side on one row
    float scale;
    uint32_t* error;
};

// a looked-up vector, scaled (zeros where the index is outside the table)
template <typename T, int VEC>
__device__ __forceinline__ void emb_scaled(const EmbArgs& E, int64_t at, bool live, const EmbVec<T, VEC>& x) {
    float f[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) f[k] = live ? emb_float(x.v[k]) * E.scale : 0.0f;
    emb_store<VEC>(E.out, at, E.out_type, f);
}

// Rows of more than a vector per lane: a group of lanes per row, four vectors a lane in flight.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) embedding_kernel(EmbArgs E) {
    const int lanes = 1 << E.log_lanes;
    const int lane = threadIdx.x & (lanes - 1);
    const int64_t first = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> E.log_lanes;
    const int64_t step = ((int64_t)gridDim.x * 256) >> E.log_lanes;
    const T* table = static_cast<const T*>(E.table);
    bool bad = false;
    for (int64_t t = first; t < E.tokens; t += step) {
        const int64_t i = emb_index(E.index, E.index64, t);
        const bool live = i >= 0 && i < E.rows;
        bad |= !live;
        const T* src = table + (live ? i : 0) * E.ldt;
        for (int64_t c0 = (int64_t)lane * VEC; c0 < E.width; c0 += (int64_t)lanes * VEC * 4) {
            EmbVec<T, VEC> x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int64_t c = c0 + (int64_t)u * lanes * VEC;
                if (live && c < E.width) x[u] = *reinterpret_cast<const EmbVec<T, VEC>*>(src + c);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int64_t c = c0 + (int64_t)u * lanes * VEC;
                if (c < E.width) emb_scaled<T, VEC>(E, t * E.width + c, live, x[u]);
            }
        }
    }
    if (bad && lane == 0) emb_bad_index(E.error);
}

// Rows of at most a vector per lane: eight rows a group in flight, indices first.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) embedding_rows_kernel(EmbArgs E) {
    const int lanes = 1 << E.log_lanes, groups = 256 >> E.log_lanes;
    const int lane = threadIdx.x & (lanes - 1), group = threadIdx.x >> E.log_lanes;
    const int64_t c = (int64_t)lane * VEC;
    const bool in = c < E.width;
    const T* table = static_cast<const T*>(E.table);
    bool bad = false;
    for (int64_t t0 = (int64_t)blockIdx.x * groups * 8; t0 < E.tokens; t0 += (int64_t)gridDim.x * groups * 8) {
        int64_t i[8];
        EmbVec<T, VEC> x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int64_t t = t0 + u * groups + group;
            i[u] = t < E.tokens ? emb_index(E.index, E.index64, t) : 0;
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int64_t t = t0 + u * groups + group;
            if (i[u] < 0 || i[u] >= E.rows) {
                bad |= t < E.tokens;
                i[u] = -1;
            } else if (in && t < E.tokens) {
                x[u] = *reinterpret_cast<const EmbVec<T, VEC>*>(table + i[u] * E.ldt + c);
            }
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int64_t t = t0 + u * groups + group;
            if (in && t < E.tokens) emb_scaled<T, VEC>(E, t * E.width + c, i[u] >= 0, x[u]);
        }
    }
    if (bad && lane == 0) emb_bad_index(E.error);
}

// ---------------------------------------------------------------- backward

struct EmbGradArgs {
    int64_t tokens, rows, width, ldg, ldo;
    const void* grad;
    const void* index;
    int index64;
    int64_t padding;     // -1: none
    void* out;
    int out_type, accumulate;
    float scale;
    uint32_t* error;
    // plan
    int passes, bits;    // radix passes and digit bits
    int parts, kpt;      // sorting blocks, keys per thread and tile
    int64_t part_tokens; // tokens a sorting block owns
    int lanes;           // lanes of a worker
    int tiles;           // column tiles of lanes * VEC
    int64_t share;       // sorted tokens of one worker's task
    int64_t shares;
    int zero_first;      // the whole table zeroed beside the sort; else its absent rows after it
    // workspace
    uint32_t* barrier;
    uint32_t* counts;    // [bins][parts], then their scans
    uint32_t* totals;    // [bins]
    uint32_t* key[2];
    int32_t* pos[2];
    float* part_sums;    // [shares][2][width]
};

// Arrivals of `blocks` blocks counted in one word (E.barrier[0]: the whole grid, [1]: the sorting
// blocks); the kernel is launched cooperatively, so every block runs.  A wait that runs out sets its bit of
// the error word and lets its block go on to the end of the kernel without touching the output.
__device__ __forceinline__ bool emb_sync(const EmbGradArgs& E, int word, uint32_t blocks, uint32_t& target) {
    if (blocks == 1) {
        __syncthreads();
        return true;
    }
    __shared__ int ok_s;
    target += blocks;
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        uint32_t seen = atomicAdd(E.barrier + word, 1u) + 1u;
        uint32_t i = 0;
        while ((int32_t)(seen - target) < 0 && i < EMB_WAIT_TRIES) {
            asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(E.barrier + word) : "memory");
            ++i;
        }
        const int ok = (int32_t)(seen - target) >= 0;
        if (!ok) atomicOr(E.error, EMB_GAVE_UP);
        __threadfence();
        ok_s = ok;
    }
    __syncthreads();
    return ok_s != 0;
}

// token t's sort key: its row, or `rows` (sorted last, no gradient) for the padding index and for an
// index outside the table
__device__ __forceinline__ uint32_t emb_key(const EmbGradArgs& E, int64_t t) {
    const int64_t i = emb_index(E.index, E.index64, t);
    if (i < 0 || i >= E.rows) {
        emb_bad_index(E.error);
        return (uint32_t)E.rows;
    }
    return i == E.padding ? (uint32_t)E.rows : (uint32_t)i;
}

struct EmbSortShared {
    uint32_t base[EMB_BINS];                  // next position of each digit for this block
    uint16_t warp_count[EMB_WARPS][EMB_BINS];
    uint32_t scan[EMB_WARPS];
};

// exclusive scan over the block's 512 threads
__device__ __forceinline__ uint32_t emb_block_scan(uint32_t v, uint32_t* warp_sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    uint32_t before = 0;
    for (int w = 0; w < warp; ++w) before += warp_sums[w];
    __syncthreads();
    return before + x - v;
}

// one radix pass of the calling (sorting) block's range; false when a barrier gave up
__device__ bool emb_radix_pass(const EmbGradArgs& E, int pass, uint32_t& target, EmbSortShared& S) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int shift = pass * E.bits, bins = 1 << E.bits;
    const uint32_t mask = (uint32_t)bins - 1u;
    const int64_t lo = (int64_t)blockIdx.x * E.part_tokens;
    const int64_t hi = lo + E.part_tokens < E.tokens ? lo + E.part_tokens : E.tokens;
    const uint32_t* src_key = E.key[(pass & 1) ^ 1];
    const int32_t* src_pos = E.pos[(pass & 1) ^ 1];
    {
        for (int b = threadIdx.x; b < bins; b += EMB_THREADS) S.base[b] = 0;
        __syncthreads();
        for (int64_t t0 = lo; t0 < hi; t0 += EMB_THREADS) {
            const int64_t t = t0 + threadIdx.x;
            const bool live = t < hi;
            const uint32_t digit = live ? (((pass ? __ldcg(src_key + t) : emb_key(E, t)) >> shift) & mask) : EMB_BINS;
            const uint32_t peers = __match_any_sync(0xffffffffu, digit);
            if (live && (peers & ((1u << lane) - 1u)) == 0) atomicAdd(&S.base[digit], (uint32_t)__popc(peers));
        }
        __syncthreads();
    }
    if (E.parts == 1) {  // the block's own counts are the totals
        const uint32_t v = threadIdx.x < bins ? S.base[threadIdx.x] : 0;
        const uint32_t x = emb_block_scan(v, S.scan);
        if (threadIdx.x < bins) S.base[threadIdx.x] = x;
        __syncthreads();
    } else {
        for (int b = threadIdx.x; b < bins; b += EMB_THREADS) E.counts[(int64_t)b * E.parts + blockIdx.x] = S.base[b];
        if (!emb_sync(E, 1, E.parts, target)) return false;
        for (int b = blockIdx.x * EMB_WARPS + warp; b < bins; b += E.parts * EMB_WARPS) {
            uint32_t run = 0;
            for (int p0 = 0; p0 < E.parts; p0 += 32) {
                const int p = p0 + lane;
                const uint32_t v = p < E.parts ? __ldcg(E.counts + (int64_t)b * E.parts + p) : 0;
                uint32_t x = v;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
                    if (lane >= o) x += y;
                }
                if (p < E.parts) E.counts[(int64_t)b * E.parts + p] = run + x - v;
                run += __shfl_sync(0xffffffffu, x, 31);
            }
            if (lane == 0) E.totals[b] = run;
        }
        if (!emb_sync(E, 1, E.parts, target)) return false;
        const uint32_t v = threadIdx.x < bins ? __ldcg(E.totals + threadIdx.x) : 0;
        const uint32_t x = emb_block_scan(v, S.scan);
        if (threadIdx.x < bins) S.base[threadIdx.x] = x + __ldcg(E.counts + (int64_t)threadIdx.x * E.parts + blockIdx.x);
        __syncthreads();
    }
    {
        uint32_t* dst_key = E.key[pass & 1];
        int32_t* dst_pos = E.pos[pass & 1];
        const int64_t tile = (int64_t)EMB_THREADS * E.kpt;
        for (int64_t t0 = lo; t0 < hi; t0 += tile) {
            for (int b = lane; b < bins; b += 32) S.warp_count[warp][b] = 0;
            __syncwarp();
            uint32_t key[EMB_MAX_KPT];
            int32_t pos[EMB_MAX_KPT];
            uint16_t rank[EMB_MAX_KPT];
            const int64_t w0 = t0 + (int64_t)warp * 32 * E.kpt;  // a warp's keys are consecutive
#pragma unroll
            for (int k = 0; k < EMB_MAX_KPT; ++k) {
                const int64_t t = w0 + k * 32 + lane;
                const bool live = k < E.kpt && t < hi;
                key[k] = live ? (pass ? __ldcg(src_key + t) : emb_key(E, t)) : 0;
                pos[k] = live ? (pass ? __ldcg(src_pos + t) : (int32_t)t) : -1;
            }
#pragma unroll
            for (int k = 0; k < EMB_MAX_KPT; ++k) {
                if (k < E.kpt) {
                    const uint32_t digit = pos[k] >= 0 ? ((key[k] >> shift) & mask) : EMB_BINS;
                    const uint32_t peers = __match_any_sync(0xffffffffu, digit);
                    const uint32_t below = peers & ((1u << lane) - 1u);
                    const uint16_t old = digit < EMB_BINS ? S.warp_count[warp][digit] : 0;
                    __syncwarp();
                    if (digit < EMB_BINS && below == 0) S.warp_count[warp][digit] = (uint16_t)(old + __popc(peers));
                    __syncwarp();
                    rank[k] = (uint16_t)(old + __popc(below));
                }
            }
            __syncthreads();
            uint32_t next = 0;
            if (threadIdx.x < bins) {  // counts of the warps before, per digit
                uint32_t run = 0;
                for (int w = 0; w < EMB_WARPS; ++w) {
                    const uint16_t c = S.warp_count[w][threadIdx.x];
                    S.warp_count[w][threadIdx.x] = (uint16_t)run;
                    run += c;
                }
                next = run;
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < EMB_MAX_KPT; ++k) {
                if (k < E.kpt && pos[k] >= 0) {
                    const uint32_t digit = (key[k] >> shift) & mask;
                    const uint32_t at = S.base[digit] + S.warp_count[warp][digit] + rank[k];
                    dst_key[at] = key[k];
                    dst_pos[at] = pos[k];
                }
            }
            __syncthreads();
            if (threadIdx.x < bins) S.base[threadIdx.x] += next;
            __syncthreads();
        }
    }
    return pass + 1 == E.passes || emb_sync(E, 1, E.parts, target);
}

__device__ __forceinline__ int64_t emb_lower_bound(const uint32_t* key, int64_t n, uint32_t v) {
    int64_t lo = 0;
    while (n > 0) {
        const int64_t half = n >> 1;
        if (__ldcg(key + lo + half) < v) {
            lo += half + 1;
            n -= half + 1;
        } else {
            n = half;
        }
    }
    return lo;
}

// a finished row: rounded once, or added to what the table's gradient holds and rounded once
template <int VEC>
__device__ __forceinline__ void emb_finish(const EmbGradArgs& E, uint32_t row, int64_t c, float* sum) {
    const int64_t at = (int64_t)row * E.ldo + c;
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum[i] *= E.scale;
    if (E.accumulate) {
        float old[VEC];
        emb_load_typed<VEC>(E.out, at, E.out_type, old);
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum[i] += old[i];
    }
    emb_store<VEC>(E.out, at, E.out_type, sum);
}

template <int VEC>
__device__ __forceinline__ void emb_part(float* part_sums, int64_t share, int slot, int64_t width, int64_t c,
                                         const float* sum) {
    emb_store<VEC>(part_sums, (share * 2 + slot) * width + c, EMB_F32, sum);
}

template <int VEC>
__device__ __forceinline__ void emb_zero_row(const EmbGradArgs& E, int64_t row, int lane, int lanes) {
    float zero[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) zero[i] = 0.0f;
    for (int64_t c = (int64_t)lane * VEC; c < E.width; c += (int64_t)lanes * VEC)
        emb_store<VEC>(E.out, row * E.ldo + c, E.out_type, zero);
}

__device__ __forceinline__ uint32_t emb_last_key(const EmbGradArgs& E, const uint32_t* key, int64_t share) {
    const int64_t end = (share + 1) * E.share;
    return __ldcg(key + (end < E.tokens ? end : E.tokens) - 1);
}

// parts of the run that starts in `share` and goes on past its end; 0 where there is none.  The lanes of a
// worker (in step) look at the first keys of as many shares after it at once, in strides that grow while all of
// them belong to the run and shrink again where it ends: of 83,414 x 8 tokens' rows, Zipf-distributed over 1,331,
// the longest run crosses hundreds of shares; looked at one group after another they took half of the 84 us.
__device__ __forceinline__ int64_t emb_run_parts(const EmbGradArgs& E, const uint32_t* key, int64_t share, int lane, int lanes,
                                                 uint32_t group_mask) {
    const int64_t begin = share * E.share, end = begin + E.share;
    if (end >= E.tokens) return 0;
    const uint32_t run = __ldcg(key + end - 1), next = __ldcg(key + end);
    const uint32_t before = begin > 0 ? __ldcg(key + begin - 1) : 0xffffffffu;
    if (run >= (uint32_t)E.rows || next != run || before == run) return 0;
    int64_t last = 1, stride = 1;
    bool up = true;
    while (up || stride > 1) {
        if (!up) stride /= lanes;
        const int64_t at = (share + last + (lane + 1) * stride) * E.share;
        const uint32_t on = __ballot_sync(group_mask, at < E.tokens && __ldcg(key + at) == run) & group_mask;
        const int more = __popc(on);  // sorted keys: the shares that the run reaches come first
        last += more * stride;
        if (up && more == lanes) stride *= lanes;
        else up = false;
    }
    return last + 1;
}

// parts [i0, i1) of the run that starts in `share`: part 0 is that share's tail, part i the head of the
// i-th share after it
template <int VEC>
__device__ __forceinline__ void emb_sum_parts(const EmbGradArgs& E, int64_t share, int64_t c, int64_t i0, int64_t i1,
                                              float* sum) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) sum[k] = 0.0f;
    for (int64_t i = i0; i < i1; i += 4) {
        float x[4][VEC];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (i + u < i1) {
                const float* p = E.part_sums + ((share + i + u) * 2 + (i + u == 0 ? 1 : 0)) * E.width + c;
                if constexpr (VEC >= 4) {
#pragma unroll
                    for (int q = 0; q < VEC / 4; ++q) {
                        const float4 f = __ldcg(reinterpret_cast<const float4*>(p) + q);
                        x[u][4 * q] = f.x, x[u][4 * q + 1] = f.y, x[u][4 * q + 2] = f.z, x[u][4 * q + 3] = f.w;
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < VEC; ++k) x[u][k] = __ldcg(p + k);
                }
            } else {
#pragma unroll
                for (int k = 0; k < VEC; ++k) x[u][k] = 0.0f;
            }
        }
#pragma unroll
        for (int k = 0; k < VEC; ++k) sum[k] += (x[0][k] + x[1][k]) + (x[2][k] + x[3][k]);
    }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(EMB_THREADS, 2) embedding_backward_kernel(EmbGradArgs E) {
    __shared__ EmbSortShared S;
    const int lane32 = threadIdx.x & 31;
    const int64_t warps = (int64_t)gridDim.x * EMB_WARPS;
    const int64_t gwarp = (int64_t)blockIdx.x * EMB_WARPS + (threadIdx.x >> 5);
    uint32_t target = 0, sort_target = 0;

    if (E.zero_first && !(E.parts < (int)gridDim.x && (int)blockIdx.x < E.parts)) {
        // the blocks that do not sort zero the table meanwhile (all of them where every block sorts)
        const int64_t skip = E.parts < (int)gridDim.x ? E.parts : 0, blocks = gridDim.x - skip, block = blockIdx.x - skip;
        const int64_t bytes = E.rows * E.width * (E.out_type == EMB_F32 ? 4 : 2);
        if ((E.ldo == E.width || E.rows == 1) && ((uintptr_t)E.out & 15) == 0) {
            uint4* out = static_cast<uint4*>(E.out);
#pragma unroll 8
            for (int64_t i = block * EMB_THREADS + threadIdx.x; i < bytes / 16; i += blocks * EMB_THREADS) out[i] = make_uint4(0u, 0u, 0u, 0u);
            if (block == 0 && threadIdx.x < bytes % 16) static_cast<unsigned char*>(E.out)[bytes / 16 * 16 + threadIdx.x] = 0;
        } else {
            for (int64_t r = block * EMB_WARPS + (threadIdx.x >> 5); r < E.rows; r += blocks * EMB_WARPS) emb_zero_row<VEC>(E, r, lane32, 32);
        }
    }
    if ((int)blockIdx.x < E.parts)
        for (int pass = 0; pass < E.passes; ++pass)
            if (!emb_radix_pass(E, pass, sort_target, S)) return;
    if (!emb_sync(E, 0, gridDim.x, target)) return;
    const uint32_t* key = E.key[(E.passes & 1) ^ 1];
    const int32_t* pos = E.pos[(E.passes & 1) ^ 1];
    const uint32_t rows = (uint32_t)E.rows;

    // ------------------------------------------------ segment sums
    constexpr int U = sizeof(T) * VEC == 16 ? 4 : 8;  // rows in flight per worker: 64 KB or less an SM
    const int lanes = E.lanes, lane = threadIdx.x & (lanes - 1);
    const int64_t workers = warps * (32 / lanes);
    const int64_t worker = ((int64_t)blockIdx.x * EMB_THREADS + threadIdx.x) / lanes;
    const uint32_t group_mask = lanes == 32 ? 0xffffffffu : (((1u << lanes) - 1u) << (lane32 & ~(lanes - 1)));
    const T* grad = static_cast<const T*>(E.grad);
    const int64_t tasks = E.shares * E.tiles;
    for (int64_t task = worker; task < tasks; task += workers) {
        const int64_t share = task % E.shares;
        const int64_t c = (task / E.shares) * ((int64_t)lanes * VEC) + (int64_t)lane * VEC;
        const bool in = c < E.width;
        const int64_t begin = share * E.share;
        const int64_t end = begin + E.share < E.tokens ? begin + E.share : E.tokens;
        uint32_t run = __ldcg(key + begin);
        bool head = begin > 0 && __ldcg(key + begin - 1) == run;  // the run started in an earlier share
        float sum[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum[i] = 0.0f;
        for (int64_t e0 = begin; e0 < end; e0 += U) {
            // lane j of the worker fetches entry j
            const int64_t mine = e0 + (lane & (U - 1));
            const uint32_t my_key = mine < end ? __ldcg(key + mine) : rows;
            const int32_t my_pos = mine < end ? __ldcg(pos + mine) : 0;
            const int n = end - e0 < U ? (int)(end - e0) : U;
            EmbVec<T, VEC> x[U];  // as loaded: converted where they are added
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const uint32_t k = __shfl_sync(group_mask, my_key, j, lanes);
                const int64_t p = __shfl_sync(group_mask, my_pos, j, lanes);
                if (in && k < rows) {
                    x[j] = *reinterpret_cast<const EmbVec<T, VEC>*>(grad + p * E.ldg + c);
                } else {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) x[j].v[i] = emb_zero<T>();
                }
            }
            const uint32_t first = __shfl_sync(group_mask, my_key, 0, lanes);
            const uint32_t last = __shfl_sync(group_mask, my_key, U - 1, lanes);
            if (n == U && first == run && last == run) {  // all of the same run: a tree
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    float four[U / 4];
#pragma unroll
                    for (int q = 0; q < U / 4; ++q)
                        four[q] = (emb_float(x[4 * q].v[i]) + emb_float(x[4 * q + 1].v[i])) +
                                  (emb_float(x[4 * q + 2].v[i]) + emb_float(x[4 * q + 3].v[i]));
                    sum[i] += U == 8 ? four[0] + four[U / 4 - 1] : four[0];
                }
                continue;
            }
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const uint32_t k = __shfl_sync(group_mask, my_key, j, lanes);
                if (j < n) {
                    if (k != run) {
                        if (in && run < rows) {
                            if (head) emb_part<VEC>(E.part_sums, share, 0, E.width, c, sum);
                            else emb_finish<VEC>(E, run, c, sum);
                        }
                        run = k;
                        head = false;
#pragma unroll
                        for (int i = 0; i < VEC; ++i) sum[i] = 0.0f;
                    }
#pragma unroll
                    for (int i = 0; i < VEC; ++i) sum[i] += emb_float(x[j].v[i]);
                }
            }
        }
        if (in && run < rows) {
            const bool on = end < E.tokens && __ldcg(key + end) == run;
            if (head) emb_part<VEC>(E.part_sums, share, 0, E.width, c, sum);
            else if (on) emb_part<VEC>(E.part_sums, share, 1, E.width, c, sum);
            else emb_finish<VEC>(E, run, c, sum);
        }
    }
    // rows that no token has
    if (!E.accumulate && !E.zero_first) {
        for (int64_t r0 = gwarp * 32; r0 < E.rows; r0 += warps * 32) {
            const int64_t r = r0 + lane32;
            bool absent = false;
            if (r < E.rows) {
                const int64_t at = emb_lower_bound(key, E.tokens, (uint32_t)r);
                absent = at >= E.tokens || __ldcg(key + at) != (uint32_t)r;
            }
            uint32_t todo = __ballot_sync(0xffffffffu, absent);
            while (todo) {
                const int b = __ffs(todo) - 1;
                todo &= todo - 1;
                emb_zero_row<VEC>(E, r0 + b, lane32, 32);
            }
        }
    }
    if (E.shares <= 1) return;
    if (!emb_sync(E, 0, gridDim.x, target)) return;

    // ------------------------------------------------ runs that cross shares
    // The worker of the share where such a run starts adds its parts in order; a run of more than
    // EMB_SERIAL_PARTS parts is left to its whole block, whose workers add a stretch of parts each.
    __shared__ float fold[EMB_THREADS * VEC];
    __shared__ int long_count;
    __shared__ int64_t long_task[EMB_THREADS / 8];
    const int groups = EMB_THREADS / lanes, group = threadIdx.x / lanes;
    for (int64_t task0 = worker - group; task0 < tasks; task0 += workers) {
        if (threadIdx.x == 0) long_count = 0;
        __syncthreads();
        int64_t count = 0;
        if (task0 + group < tasks) {
            count = emb_run_parts(E, key, (task0 + group) % E.shares, lane, lanes, group_mask);
            if (count > EMB_SERIAL_PARTS && lane == 0) long_task[atomicAdd(&long_count, 1)] = task0 + group;
        }
        if (count > 0 && count <= EMB_SERIAL_PARTS) {
            const int64_t share = (task0 + group) % E.shares;
            const int64_t c = ((task0 + group) / E.shares) * ((int64_t)lanes * VEC) + (int64_t)lane * VEC;
            if (c < E.width) {
                float sum[VEC];
                emb_sum_parts<VEC>(E, share, c, 0, count, sum);
                emb_finish<VEC>(E, emb_last_key(E, key, share), c, sum);
            }
        }
        __syncthreads();
        for (int i = 0; i < long_count; ++i) {
            const int64_t share = long_task[i] % E.shares;
            const int64_t c = (long_task[i] / E.shares) * ((int64_t)lanes * VEC) + (int64_t)lane * VEC;
            const int64_t parts = emb_run_parts(E, key, share, lane, lanes, group_mask);
            const int64_t each = (parts + groups - 1) / groups;
            const int64_t i0 = (int64_t)group * each;
            float sum[VEC];
#pragma unroll
            for (int k = 0; k < VEC; ++k) sum[k] = 0.0f;
            if (c < E.width && i0 < parts) emb_sum_parts<VEC>(E, share, c, i0, i0 + each < parts ? i0 + each : parts, sum);
            __syncthreads();
#pragma unroll
            for (int k = 0; k < VEC; ++k) fold[k * EMB_THREADS + threadIdx.x] = sum[k];
            __syncthreads();
            if (group == 0 && c < E.width) {
                for (int g = 1; g < groups; ++g) {
#pragma unroll
                    for (int k = 0; k < VEC; ++k) sum[k] += fold[k * EMB_THREADS + g * lanes + lane];
                }
                emb_finish<VEC>(E, emb_last_key(E, key, share), c, sum);
            }
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- few tokens

// A block per row (of up to eight an SM) looks through up to this many tokens.  Measured, this way and what else
// would be taken: 4,096 tokens into 40 x 32 6.4 and 8.5 us, into 300 x 128 7.8 and 25, into 1,184 x 16 13 and 75,
// but into 4 x 32 12.5 and 7.4; 16,384 into 40 x 32 18 and 8.7, into 1,184 x 128 39 and 45; 4,096 into 2,400 x 512
// (9,600 blocks) 84 and 45 us.
constexpr int EMB_SCAN_TOKENS = 4096;
constexpr int EMB_SCAN_WARP = 256;     // up to here a warp per table row

// the rows of the tokens in `match` (bits of tokens t0 ..), added in order, eight in flight
template <typename T, int VEC>
__device__ __forceinline__ void emb_add_matches(const EmbGradArgs& E, uint32_t match, int64_t t0, int64_t c, bool in, float* sum) {
    const T* grad = static_cast<const T*>(E.grad);
    while (match) {
        EmbVec<T, VEC> x[8];
        int n = 0;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if (match) {
                const int64_t t = t0 + __ffs(match) - 1;
                match &= match - 1;
                if (in) x[u] = *reinterpret_cast<const EmbVec<T, VEC>*>(grad + t * E.ldg + c);
                n = u + 1;
            }
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if (u < n && in) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) sum[i] += emb_float(x[u].v[i]);
            }
        }
    }
}

// a warp per table row (in turn) and, where few rows leave warps idle, stretch of its columns (gridDim.y); all
// indices in its lanes
template <typename T, int VEC>
__global__ void __launch_bounds__(256) embedding_backward_warp_kernel(EmbGradArgs E) {
    const int lane = threadIdx.x & 31;
    constexpr int K = EMB_SCAN_WARP / 32;
    uint32_t key[K];
#pragma unroll
    for (int k = 0; k < K; ++k) key[k] = k * 32 + lane < E.tokens ? emb_key(E, k * 32 + lane) : 0xffffffffu;
    for (int64_t r = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5; r < E.rows; r += (int64_t)gridDim.x * 8) {
        uint32_t match[K], any = 0;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            match[k] = k * 32 < E.tokens ? __ballot_sync(0xffffffffu, key[k] == (uint32_t)r) : 0u;
            any |= match[k];
        }
        if (!any && E.accumulate) continue;
        for (int64_t c = ((int64_t)blockIdx.y * 32 + lane) * VEC; c - lane * VEC < E.width; c += (int64_t)gridDim.y * 32 * VEC) {
            const bool in = c < E.width;
            float sum[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) sum[i] = 0.0f;
            if (any) {
#pragma unroll
                for (int k = 0; k < K; ++k) emb_add_matches<T, VEC>(E, match[k], k * 32, c, in, sum);
            }
            if (in) emb_finish<VEC>(E, (uint32_t)r, c, sum);
        }
    }
}

// a block per table row and column tile: each warp a stretch of the indices, the warps' sums added in order
template <typename T, int VEC>
__global__ void __launch_bounds__(EMB_THREADS) embedding_backward_block_kernel(EmbGradArgs E) {
    __shared__ float part[EMB_WARPS][32 * VEC];
    __shared__ int any_s;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t r = blockIdx.x, c = (int64_t)blockIdx.y * 32 * VEC + (int64_t)lane * VEC;
    const bool in = c < E.width;
    const int64_t each = ((E.tokens + EMB_WARPS - 1) / EMB_WARPS + 31) & ~31ll;
    const int64_t lo = warp * each, hi = lo + each < E.tokens ? lo + each : E.tokens;
    if (threadIdx.x == 0) any_s = 0;
    __syncthreads();
    float sum[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum[i] = 0.0f;
    bool any = false;
    for (int64_t t0 = lo; t0 < hi; t0 += 32) {
        const uint32_t key = t0 + lane < hi ? emb_key(E, t0 + lane) : 0xffffffffu;
        const uint32_t match = __ballot_sync(0xffffffffu, key == (uint32_t)r);
        any |= match != 0;
        emb_add_matches<T, VEC>(E, match, t0, c, in, sum);
    }
    if (any) any_s = 1;
#pragma unroll
    for (int i = 0; i < VEC; ++i) part[warp][i * 32 + lane] = sum[i];
    __syncthreads();
    if (warp == 0 && in && (any_s || !E.accumulate)) {
        for (int w = 1; w < EMB_WARPS; ++w) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) sum[i] += part[w][i * 32 + lane];
        }
        emb_finish<VEC>(E, (uint32_t)r, c, sum);
    }
}

// ---------------------------------------------------------------- few table rows

constexpr int EMB_TABLE_BYTES = 104 * 1024;  // a block's tables: two blocks fit an SM
constexpr int EMB_TABLE_ROWS = 52;           // at most: four warps' tables of 128 columns

// grid (blocks, column tiles); E.parts warps a block; tables [warp][row][32 lanes x VEC]
template <typename T, int VEC>
__global__ void __launch_bounds__(EMB_THREADS, 2) embedding_backward_table_kernel(EmbGradArgs E) {
    extern __shared__ __align__(16) float emb_tables[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = E.parts;
    const int rows = (int)E.rows;
    const int64_t c = (int64_t)blockIdx.y * 32 * VEC + (int64_t)lane * VEC;
    const bool in = c < E.width;
    const T* grad = static_cast<const T*>(E.grad);
    EmbVec<float, VEC>* table = reinterpret_cast<EmbVec<float, VEC>*>(emb_tables) + (size_t)warp * rows * 32 + lane;
    EmbVec<float, VEC> zero;
#pragma unroll
    for (int i = 0; i < VEC; ++i) zero.v[i] = 0.0f;
    for (int r = 0; r < rows; ++r) table[r * 32] = zero;
    // each warp a contiguous stretch
    const int64_t lo = ((int64_t)blockIdx.x * warps + warp) * E.share, hi = lo + E.share < E.tokens ? lo + E.share : E.tokens;
    for (int64_t t0 = lo; t0 < hi; t0 += 32) {
        const uint32_t my_key = t0 + lane < hi ? emb_key(E, t0 + lane) : (uint32_t)rows;
        const int n = hi - t0 < 32 ? (int)(hi - t0) : 32;
#pragma unroll
        for (int j0 = 0; j0 < 32; j0 += 8) {
            if (j0 >= n) break;
            EmbVec<T, VEC> x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t k = __shfl_sync(0xffffffffu, my_key, j0 + j);
                if (in && k < (uint32_t)rows) x[j] = *reinterpret_cast<const EmbVec<T, VEC>*>(grad + (t0 + j0 + j) * E.ldg + c);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t k = __shfl_sync(0xffffffffu, my_key, j0 + j);
                if (k < (uint32_t)rows) {
                    EmbVec<float, VEC> f = table[k * 32];
                    if (in) {
#pragma unroll
                        for (int i = 0; i < VEC; ++i) f.v[i] += emb_float(x[j].v[i]);
                    }
                    table[k * 32] = f;
                }
            }
        }
    }
    __syncthreads();
    // the warps' tables in order -> this block's, [block][row][width]
    for (int r = warp; r < rows; r += warps) {
        EmbVec<float, VEC> f = zero;
        for (int w = 0; w < warps; ++w) {
            const EmbVec<float, VEC> g = reinterpret_cast<EmbVec<float, VEC>*>(emb_tables)[((size_t)w * rows + r) * 32 + lane];
#pragma unroll
            for (int i = 0; i < VEC; ++i) f.v[i] += g.v[i];
        }
        if (in) emb_store<VEC>(E.part_sums, ((int64_t)blockIdx.x * rows + r) * E.width + c, EMB_F32, f.v);
    }
}

// few blocks' tables in order: a column a thread.  Measured, with this fold and with the next: 9,000 tokens into
// 30,000 x 16 (5 tables) 14.4 and 44 us, 50,000 into 8,000 x 8 (25) 17.6 and 20.7, 100,000 into 10,000 x 2 (49)
// 20.7 and 18.5, 500,000 into 1,024 x 1 (245) 48 and 33 us; where few sums leave both a few us, they are alike.
constexpr int EMB_FOLD_FEW = 32;
__global__ void __launch_bounds__(256) embedding_backward_fold_few_kernel(EmbGradArgs E, int blocks) {
    const int64_t total = E.rows * E.width, at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= total) return;
    float sum = 0.0f;
    for (int b = 0; b < blocks; b += 8) {
        float x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) x[u] = b + u < blocks ? __ldcg(E.part_sums + (int64_t)(b + u) * total + at) : 0.0f;
        sum += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
    }
    if (sum != 0.0f || !E.accumulate) emb_finish<1>(E, (uint32_t)(at / E.width), at % E.width, &sum);
}

// the blocks' tables in order: 32 columns and 16 stretches of the blocks a block
__global__ void __launch_bounds__(EMB_THREADS) embedding_backward_fold_kernel(EmbGradArgs E, int blocks) {
    __shared__ float part[EMB_WARPS][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t total = E.rows * E.width, at = (int64_t)blockIdx.x * 32 + lane;
    const int each = (blocks + EMB_WARPS - 1) / EMB_WARPS, lo = warp * each, hi = lo + each < blocks ? lo + each : blocks;
    float sum = 0.0f;
    if (at < total) {
        for (int b = lo; b < hi; b += 4) {
            float x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) x[u] = b + u < hi ? __ldg(E.part_sums + (int64_t)(b + u) * total + at) : 0.0f;
            sum += (x[0] + x[1]) + (x[2] + x[3]);
        }
    }
    part[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && at < total) {
        for (int w = 1; w < EMB_WARPS; ++w) sum += part[w][lane];
        if (sum != 0.0f || !E.accumulate) emb_finish<1>(E, (uint32_t)(at / E.width), at % E.width, &sum);
    }
}

// ---------------------------------------------------------------- narrow rows

// A block keeps the fp32 sums of a range of table rows and up to 16 columns in shared memory; each of its warps
// owns the rows of one residue class of them, so that every row has one writer.  grid (shares of the tokens,
// row ranges, column tiles).
constexpr int EMB_NARROW_COLS = 16;           // a token's row in a lane's registers
constexpr int EMB_NARROW_FLOATS = 22 * 1024;  // of sums: two blocks fit an SM
constexpr int EMB_NARROW_CHUNK = 2048;        // tokens looked through at a time
constexpr int EMB_NARROW_QUEUE = 96;          // of a warp: two batches of 32 are added at once, 32 more may come
constexpr int EMB_NARROW_SHARE = 1024;        // tokens of a share at least
constexpr int EMB_NARROW_BIG = 6;             // lanes of a batch on one row, from which they add across lanes
constexpr int EMB_NARROW_ROWS = 1024;         // of the table at least
constexpr int64_t EMB_NARROW_LOOKS = 720000;  // blocks that divide the table x tokens, at most
constexpr int EMB_NARROW_SMEM = 4 * (EMB_NARROW_FLOATS + EMB_NARROW_CHUNK + 2 * EMB_WARPS * EMB_NARROW_QUEUE);

struct EmbNarrow {
    int cols, stride;   // of a column tile, and of a row's sums in shared memory: odd, for the banks
    int64_t rows;       // of a range
    int64_t ranges, tiles, shares, share;
};

// one token a lane (row: its row in the range, or -1) added to the warp's rows, in the order of the lanes
__device__ __forceinline__ void emb_narrow_add(float* table, int cols, int stride, int row, const float* v, int lane) {
    const uint32_t same = __match_any_sync(0xffffffffu, row);
    bool has = row >= 0;
    // rows that many lanes have: summed across the lanes, in an order that the lanes alone determine
    for (uint32_t big; (big = __ballot_sync(0xffffffffu, has && __popc(same) >= EMB_NARROW_BIG)) != 0u;) {
        const int leader = __ffs(big) - 1;
        const uint32_t members = __shfl_sync(0xffffffffu, same, leader);
        const int r = __shfl_sync(0xffffffffu, row, leader);
        const bool in = (members >> lane) & 1u;
        // halves of the columns change lanes, then quarters and so on: a column per pair of lanes is left
        float x[EMB_NARROW_COLS];
#pragma unroll
        for (int c = 0; c < EMB_NARROW_COLS; ++c) x[c] = in && c < cols ? v[c] : 0.0f;
#pragma unroll
        for (int d = 16; d > 1; d >>= 1) {
            const bool upper = lane & d;
#pragma unroll
            for (int c = 0; c < d / 2; ++c) {
                const float give = upper ? x[c] : x[c + d / 2], keep = upper ? x[c + d / 2] : x[c];
                x[c] = keep + __shfl_xor_sync(0xffffffffu, give, d);
            }
        }
        x[0] += __shfl_xor_sync(0xffffffffu, x[0], 1);
        if (!(lane & 1) && lane / 2 < cols) table[r * stride + lane / 2] += x[0];
        if (in) has = false;
        __syncwarp();
    }
    const int turn = __popc(same & ((1u << lane) - 1u));
    for (int k = 0; __any_sync(0xffffffffu, has); ++k) {
        if (has && turn == k) {
            float* to = table + row * stride;
#pragma unroll
            for (int c = 0; c < EMB_NARROW_COLS; c += 8) {
                float x[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = c + i < cols ? to[c + i] : 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (c + i < cols) to[c + i] = x[i] + v[c + i];
            }
            has = false;
        }
        __syncwarp();
    }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(EMB_THREADS, 2) embedding_backward_narrow_kernel(EmbGradArgs E, EmbNarrow N) {
    extern __shared__ __align__(16) float emb_tables[];
    float* table = emb_tables;
    uint32_t* list = reinterpret_cast<uint32_t*>(table + EMB_NARROW_FLOATS);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t* queue_row = list + EMB_NARROW_CHUNK + warp * 2 * EMB_NARROW_QUEUE;
    uint32_t* queue_at = queue_row + EMB_NARROW_QUEUE;
    __shared__ uint32_t found[EMB_WARPS];
    const int64_t row0 = (int64_t)blockIdx.y * N.rows, c0 = (int64_t)blockIdx.z * N.cols;
    const int rows = (int)(E.rows - row0 < N.rows ? E.rows - row0 : N.rows);
    const int cols = (int)(E.width - c0 < N.cols ? E.width - c0 : N.cols);
    const int64_t lo = (int64_t)blockIdx.x * N.share, hi = lo + N.share < E.tokens ? lo + N.share : E.tokens;
    const T* grad = static_cast<const T*>(E.grad) + lo * E.ldg + c0;
    const int stride = N.stride;
    for (int i = threadIdx.x; i < rows * stride; i += EMB_THREADS) table[i] = 0.0f;
    int queued = 0;
    // the queue's first n (up to 64) tokens, both batches' rows in flight at once
    auto add = [&](int n) {
        float v[2][EMB_NARROW_COLS];
        int row[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int i = b * 32 + lane;
            row[b] = i < n ? (int)queue_row[i] : -1;
            const T* p = grad + (i < n ? (int64_t)queue_at[i] : 0) * E.ldg;
#pragma unroll
            for (int c = 0; c < EMB_NARROW_COLS; c += VEC) {
                if (row[b] >= 0 && c < cols) emb_load<T, VEC>(p + c, v[b] + c);
            }
        }
        emb_narrow_add(table, cols, stride, row[0], v[0], lane);
        if (n > 32) emb_narrow_add(table, cols, stride, row[1], v[1], lane);
    };
    constexpr int K = EMB_NARROW_CHUNK / EMB_THREADS;
    for (int64_t t0 = lo; t0 < hi; t0 += EMB_NARROW_CHUNK) {
        // the chunk's tokens of this range, in order: (row, place in the chunk); each warp looks at a stretch
        uint32_t key[K], in[K], count = 0;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int64_t t = t0 + warp * (32 * K) + k * 32 + lane;
            key[k] = t < hi ? emb_key(E, t) : 0xffffffffu;
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const bool mine = key[k] < (uint32_t)E.rows && (int64_t)key[k] >= row0 && (int64_t)key[k] < row0 + rows;
            in[k] = __ballot_sync(0xffffffffu, mine);
            count += __popc(in[k]);
        }
        __syncthreads();  // the list and the counts are free (and the table is cleared)
        if (lane == 0) found[warp] = count;
        __syncthreads();
        uint32_t at = 0, total = 0;
        for (int w = 0; w < EMB_WARPS; ++w) {
            if (w < warp) at += found[w];
            total += found[w];
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if ((in[k] >> lane) & 1u)
                list[at + __popc(in[k] & ((1u << lane) - 1u))] =
                    (uint32_t)((int64_t)key[k] - row0) * EMB_NARROW_CHUNK + warp * (32 * K) + k * 32 + lane;
            at += __popc(in[k]);
        }
        __syncthreads();
        // each warp: its rows' tokens to its queue
        for (uint32_t i0 = 0; i0 < total; i0 += 32) {
            const uint32_t entry = i0 + lane < total ? list[i0 + lane] : 0u;
            const uint32_t row = entry / EMB_NARROW_CHUNK;
            const bool mine = i0 + lane < total && (row & (EMB_WARPS - 1)) == (uint32_t)warp;
            const uint32_t who = __ballot_sync(0xffffffffu, mine);
            if (mine) {
                const int q = queued + __popc(who & ((1u << lane) - 1u));
                queue_row[q] = row;
                queue_at[q] = (uint32_t)(t0 - lo) + entry % EMB_NARROW_CHUNK;
            }
            queued += __popc(who);
            __syncwarp();
            if (queued >= 64) {
                add(64);
                queued -= 64;
                const uint32_t r = lane < queued ? queue_row[64 + lane] : 0u, a = lane < queued ? queue_at[64 + lane] : 0u;
                __syncwarp();
                if (lane < queued) queue_row[lane] = r, queue_at[lane] = a;
                __syncwarp();
            }
        }
    }
    if (queued > 0) add(queued);
    __syncthreads();
    for (int i = threadIdx.x; i < rows * cols; i += EMB_THREADS) {
        const int64_t r = row0 + i / cols, c = c0 + i % cols;
        float sum = table[i / cols * stride + i % cols];
        if (N.shares > 1) E.part_sums[((int64_t)blockIdx.x * E.rows + r) * E.width + c] = sum;
        else if (sum != 0.0f || !E.accumulate) emb_finish<1>(E, (uint32_t)r, c, &sum);
    }
}

// Whether rows are taken so, and their split.  Every block looks at its share's indices, so blocks x tokens
// bounds it; few rows leave a warp's rows to batches of one row.  Measured, sorted against this way: 9,000
// tokens into 30,000 x 16 35 and 15 us, 30,000 into 4,000 x 32 35 and 21 us, 300,000 into 4,000 x 8 54 and 41
// us; but 100,000 into 4,000 x 32 (800,000 looks) 37 and 50 us, 30,000 into 500 x 16 26 and 41 us.
static bool emb_narrow_plan(int64_t tokens, int64_t rows, int64_t width, int grid_max, EmbNarrow& N) {
    N.cols = (int)(width < EMB_NARROW_COLS ? width : EMB_NARROW_COLS);
    N.stride = N.cols | 1;
    N.tiles = (width + N.cols - 1) / N.cols;
    N.rows = EMB_NARROW_FLOATS / N.stride;
    N.ranges = (rows + N.rows - 1) / N.rows;
    N.rows = (rows + N.ranges - 1) / N.ranges;  // ranges of equal sizes
    const int64_t blocks = N.ranges * N.tiles;
    if (rows < EMB_NARROW_ROWS || blocks > EMB_NARROW_LOOKS / tokens) return false;
    int64_t most = grid_max / blocks;
    if (most > tokens / EMB_NARROW_SHARE) most = tokens / EMB_NARROW_SHARE;
    // shares by estimated microseconds: chunks looked through, then the shares' sums written and read
    double least = 0.0;
    for (int64_t shares = 1; shares == 1 || shares <= most; ++shares) {
        const int64_t share = (tokens + shares - 1) / shares, waves = (blocks * shares + grid_max - 1) / grid_max;
        const double looks = 4.0 + 3.0 * ((share + EMB_NARROW_CHUNK - 1) / EMB_NARROW_CHUNK);
        const double fold = shares > 1 ? 3.0 + (double)shares * rows * width * 8 / 4e6 : 0.0;
        const double t = waves * looks + fold;
        if (shares == 1 || t < least) least = t, N.shares = shares, N.share = share;
    }
    N.shares = (tokens + N.share - 1) / N.share;
    return true;
}

// ---------------------------------------------------------------- host

// elements of a vector access: the widest of 16 bytes that width, strides and addresses allow
static int emb_vec(int size, int64_t width, int64_t ld, const void* p, int out_size, int64_t ldo, const void* out) {
    for (int v = 16 / size; v > 1; v /= 2) {
        const int ob = v * out_size > 16 ? 16 : v * out_size;
        if (width % v == 0 && ld % v == 0 && ldo % v == 0 && (uintptr_t)p % (v * size) == 0 && (uintptr_t)out % ob == 0)
            return v;
    }
    return 1;
}

static int emb_size(int type) { return type == EMB_F32 ? 4 : 2; }

template <typename T, int VEC>
static void (*emb_forward_of(bool one))(EmbArgs) { return one ? embedding_rows_kernel<T, VEC> : embedding_kernel<T, VEC>; }
template <typename T>
static void (*emb_forward_kernel(int vec, bool one))(EmbArgs) {
    if constexpr (sizeof(T) == 2) {
        if (vec == 8) return emb_forward_of<T, 8>(one);
    }
    return vec == 4 ? emb_forward_of<T, 4>(one) : vec == 2 ? emb_forward_of<T, 2>(one) : emb_forward_of<T, 1>(one);
}

enum { EMB_SORT = 0, EMB_WARP = 1, EMB_BLOCK = 2, EMB_TABLE = 3 };
template <typename T>
static void (*emb_narrow_kernel(int vec))(EmbGradArgs, EmbNarrow) {
    if constexpr (sizeof(T) == 2) {
        if (vec == 8) return embedding_backward_narrow_kernel<T, 8>;
    }
    return vec == 4 ? embedding_backward_narrow_kernel<T, 4> : vec == 2 ? embedding_backward_narrow_kernel<T, 2>
                                                                        : embedding_backward_narrow_kernel<T, 1>;
}
template <typename T, int VEC>
static void (*emb_backward_of(int path))(EmbGradArgs) {
    if (path == EMB_WARP) return embedding_backward_warp_kernel<T, VEC>;
    if (path == EMB_BLOCK) return embedding_backward_block_kernel<T, VEC>;
    if constexpr (VEC <= 4) {
        if (path == EMB_TABLE) return embedding_backward_table_kernel<T, VEC>;
    }
    return embedding_backward_kernel<T, VEC>;
}
template <typename T>
static void (*emb_backward_kernel(int vec, int path))(EmbGradArgs) {
    if constexpr (sizeof(T) == 2) {
        if (vec == 8) return emb_backward_of<T, 8>(path);
    }
    return vec == 4 ? emb_backward_of<T, 4>(path) : vec == 2 ? emb_backward_of<T, 2>(path) : emb_backward_of<T, 1>(path);
}

struct EmbLayout {
    int64_t barrier, counts, totals, key0, key1, pos0, pos1, parts, bytes;
};

// The plan and workspace depend on sizes and the vector width alone; the workspace is sized for any
// vector width (the share count is bounded by the resident workers).
static void emb_plan(int64_t tokens, int64_t rows, int64_t width, int vec, int grid_max, EmbGradArgs& E, int& grid) {
    int key_bits = 1;
    while ((rows >> key_bits) != 0) ++key_bits;  // keys 0 .. rows (absent tokens)
    E.passes = (key_bits + 8) / 9;
    E.bits = (key_bits + E.passes - 1) / E.passes;
    // a worker's lanes: the fewest of 8, 16, 32 that cover a row, 32 for wider rows
    const int64_t vectors = (width + vec - 1) / vec;
    E.lanes = vectors <= 8 ? 8 : vectors <= 16 ? 16 : 32;
    E.tiles = (int)((vectors + E.lanes - 1) / E.lanes);
    const int64_t per_block = EMB_THREADS / E.lanes;
    // one task (a share of the tokens, a column tile) for each resident worker
    const int64_t most_shares = per_block * grid_max / E.tiles > 1 ? per_block * grid_max / E.tiles : 1;
    const int64_t share = (tokens + most_shares - 1) / most_shares;
    E.share = share < EMB_MIN_SHARE ? EMB_MIN_SHARE : (share + 7) / 8 * 8;
    E.shares = (tokens + E.share - 1) / E.share;
    // sorting blocks: one tile of a key per thread each at first, then more keys per thread; alone up to
    // four keys per thread, where grid barriers would cost more than the work that they share out
    if (tokens <= 4 * EMB_THREADS) {
        E.parts = 1;
        E.kpt = (int)((tokens + EMB_THREADS - 1) / EMB_THREADS);
        E.part_tokens = tokens;
    } else {
        const int64_t tiles = (tokens + EMB_THREADS - 1) / EMB_THREADS;
        const int64_t most = grid_max < 148 ? grid_max : 148;
        int64_t kpt = (tiles + most - 1) / most;
        E.kpt = (int)(kpt > EMB_MAX_KPT ? EMB_MAX_KPT : kpt);
        const int64_t whole = (int64_t)EMB_THREADS * E.kpt;
        const int64_t n = (tokens + whole - 1) / whole;  // tiles of kpt keys per thread
        const int64_t per = (n + most - 1) / most;
        E.part_tokens = per * whole;
        E.parts = (int)((tokens + E.part_tokens - 1) / E.part_tokens);
    }
    // zeroing beside the sort is free up to what the device writes in its time; every row twice costs more
    // than looking for the absent ones only in a large table that most tokens' rows fill
    E.zero_first = !E.accumulate && (tokens <= rows || rows * width * 4 <= (256ll << 20));
    int64_t want = (E.shares * E.tiles + per_block - 1) / per_block;
    if (want < E.parts) want = E.parts;
    if (!E.accumulate) {  // blocks for the zeroed rows: 64 KB each
        const int64_t z = (rows * width * 4) >> 16;
        if (want < z) want = z;
    }
    grid = (int)(want < grid_max ? want : grid_max);
}

static EmbLayout emb_layout(int64_t tokens, int64_t width, int grid_max) {
    EmbLayout L;
    auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
    int64_t at = 0;
    L.barrier = at, at += 256;
    L.totals = at, at += up(EMB_BINS * 4);
    L.counts = at, at += up((int64_t)EMB_BINS * 148 * 4);
    L.key0 = at, at += up(tokens * 4);
    L.key1 = at, at += up(tokens * 4);
    L.pos0 = at, at += up(tokens * 4);
    L.pos1 = at, at += up(tokens * 4);
    // two rows of sums a share; shares * tiles is at most the resident workers (and one share more), so
    // their columns are at most 8 per resident thread
    const int64_t by_tokens = (tokens + EMB_MIN_SHARE - 1) / EMB_MIN_SHARE * width;
    const int64_t by_threads = (int64_t)grid_max * EMB_THREADS * 8 + 2 * width;
    const int64_t sums = (by_tokens < by_threads ? by_tokens : by_threads) * 2;
    // a table of sums per block, grid_max / (column tiles of at most 128 columns) blocks or one
    const int64_t tables = EMB_TABLE_ROWS * ((int64_t)grid_max * 128 + width);
    // and a block's sums of narrow rows for at most grid_max blocks, where the tokens go to several shares
    const int64_t narrow = tokens >= 2 * EMB_NARROW_SHARE ? grid_max * (int64_t)EMB_NARROW_FLOATS : 0;
    const int64_t most = sums > tables ? sums : tables;
    L.parts = at, at += up((most > narrow ? most : narrow) * 4);
    L.bytes = at;
    return L;
}

// blocks of the backward kernel that one device holds at once
static int emb_grid_max() { return 2 * sm_count(); }

}  // namespace pbg

using namespace pbg;

extern "C" {

int pbg_embedding(int64_t tokens, int64_t rows, int64_t width, const void* index, int32_t index64, const void* table,
                  int32_t table_type, int64_t ldt, float scale, void* out, int32_t out_type, uint32_t* error, void* stream) {
    PBG_REQUIRE(tokens >= 0 && rows >= 0 && width >= 0, "embedding: negative size");
    PBG_REQUIRE(table_type >= 0 && table_type <= 2 && out_type >= 0 && out_type <= 2, "embedding: unknown type");
    if (tokens == 0 || width == 0) return 0;
    PBG_REQUIRE(index && out && error && (table || rows == 0), "embedding: null pointer");
    PBG_REQUIRE(ldt >= width || rows <= 1, "embedding: table row stride must be >= width");
    EmbArgs E;
    E.tokens = tokens, E.rows = rows, E.width = width, E.ldt = ldt;
    E.index = index, E.index64 = index64, E.table = table, E.out = out, E.out_type = out_type;
    E.scale = scale, E.error = error;
    const int vec = emb_vec(emb_size(table_type), width, rows > 1 ? ldt : 0, table, emb_size(out_type), width, out);
    const int64_t vectors = (width + vec - 1) / vec;
    // lanes of a row: a vector each up to a warp, then up to four vectors each, at most a block
    E.log_lanes = 0;
    while (E.log_lanes < 5 && (1LL << E.log_lanes) < vectors) ++E.log_lanes;
    while (E.log_lanes < 8 && (4LL << E.log_lanes) < vectors) ++E.log_lanes;
    const bool one = vectors <= (1LL << E.log_lanes) && tokens > (8LL << (8 - E.log_lanes)) * sm_count();  // eight rows a group fill the device
    const int64_t need = one ? ((tokens << E.log_lanes) + 2047) / 2048 : ((tokens << E.log_lanes) + 255) / 256;
    const int64_t most = (int64_t)sm_count() * 32;
    void (*kernel)(EmbArgs) = table_type == EMB_F32 ? emb_forward_kernel<float>(vec, one)
                              : table_type == EMB_BF16 ? emb_forward_kernel<__nv_bfloat16>(vec, one)
                                                       : emb_forward_kernel<__half>(vec, one);
    kernel<<<(unsigned)(need < most ? need : most), 256, 0, as_stream(stream)>>>(E);
    return launch_status("embedding");
}

int64_t pbg_embedding_backward_workspace(int64_t tokens, int64_t width) {
    if (tokens < 0 || width < 0) return PBG_EINVAL;
    return emb_layout(tokens, width, emb_grid_max()).bytes;
}

int pbg_embedding_backward(int64_t tokens, int64_t rows, int64_t width, const void* grad, int32_t grad_type, int64_t ldg,
                           const void* index, int32_t index64, int64_t padding, float scale, void* out, int32_t out_type,
                           int64_t ldo, int32_t accumulate, void* workspace, int64_t workspace_bytes, uint32_t* error,
                           void* stream) {
    PBG_REQUIRE(tokens >= 0 && rows >= 0 && width >= 0, "embedding_backward: negative size");
    PBG_REQUIRE(tokens < (1LL << 31) && rows < (1LL << 31), "embedding_backward: at most 2^31 - 1 tokens and rows");
    PBG_REQUIRE(grad_type >= 0 && grad_type <= 2 && out_type >= 0 && out_type <= 2, "embedding_backward: unknown type");
    if (rows == 0 || width == 0) return 0;
    PBG_REQUIRE(out && error, "embedding_backward: null pointer");
    PBG_REQUIRE(ldo >= width || rows == 1, "embedding_backward: out row stride must be >= width");
    PBG_REQUIRE(padding >= -1 && padding < rows, "embedding_backward: the padding index must be a row of the table");
    cudaStream_t s = as_stream(stream);
    if (tokens == 0) {
        if (accumulate) return 0;
        return cuda_status(cudaMemset2DAsync(out, (size_t)(rows == 1 ? width : ldo) * emb_size(out_type), 0,
                                             (size_t)width * emb_size(out_type), (size_t)rows, s),
                           "embedding_backward: zero table");
    }
    PBG_REQUIRE(grad && index && workspace, "embedding_backward: null pointer");
    PBG_REQUIRE(ldg >= width || tokens == 1, "embedding_backward: gradient row stride must be >= width");
    PBG_REQUIRE((uintptr_t)workspace % 256 == 0, "embedding_backward: workspace must be 256-byte aligned");
    const int grid_max = emb_grid_max();
    const EmbLayout L = emb_layout(tokens, width, grid_max);
    PBG_REQUIRE(workspace_bytes >= L.bytes, "embedding_backward: workspace too small");
    EmbGradArgs E;
    E.tokens = tokens, E.rows = rows, E.width = width, E.ldg = ldg, E.ldo = ldo;
    E.grad = grad, E.index = index, E.index64 = index64, E.padding = padding;
    E.out = out, E.out_type = out_type, E.accumulate = accumulate, E.scale = scale, E.error = error;
    const int vec = emb_vec(emb_size(grad_type), width, tokens > 1 ? ldg : 0, grad, emb_size(out_type), rows > 1 ? ldo : 0, out);
    int grid = 1;
    emb_plan(tokens, rows, width, vec, grid_max, E, grid);
    unsigned char* w = static_cast<unsigned char*>(workspace);
    E.barrier = reinterpret_cast<uint32_t*>(w + L.barrier);
    E.counts = reinterpret_cast<uint32_t*>(w + L.counts);
    E.totals = reinterpret_cast<uint32_t*>(w + L.totals);
    E.key[0] = reinterpret_cast<uint32_t*>(w + L.key0);
    E.key[1] = reinterpret_cast<uint32_t*>(w + L.key1);
    E.pos[0] = reinterpret_cast<int32_t*>(w + L.pos0);
    E.pos[1] = reinterpret_cast<int32_t*>(w + L.pos1);
    E.part_sums = reinterpret_cast<float*>(w + L.parts);
    auto of = [&](int v, int path) {
        return grad_type == EMB_F32 ? emb_backward_kernel<float>(v, path)
               : grad_type == EMB_BF16 ? emb_backward_kernel<__nv_bfloat16>(v, path) : emb_backward_kernel<__half>(v, path);
    };
    const int64_t column_tiles = (width + 32 * vec - 1) / (32 * vec);
    if (tokens <= EMB_SCAN_WARP) {
        const int64_t need = (rows + 7) / 8, most = (int64_t)sm_count() * 8;
        const int64_t x = need < most ? need : most, y = most / x < column_tiles ? most / x : column_tiles;
        of(vec, EMB_WARP)<<<dim3((unsigned)x, (unsigned)y), 256, 0, s>>>(E);
        return launch_status("embedding_backward");
    }
    // a block per row and column tile: up to a few of them per SM at once
    if (tokens <= EMB_SCAN_TOKENS && rows * column_tiles <= 8 * (int64_t)sm_count() && column_tiles < 65536) {
        of(vec, EMB_BLOCK)<<<dim3((unsigned)rows, (unsigned)column_tiles), EMB_THREADS, 0, s>>>(E);
        return launch_status("embedding_backward");
    }
    if (rows <= EMB_TABLE_ROWS && width >= 32) {
        // 32 lanes' vectors of at most 16 bytes of sums, no wider than the row
        int v = vec > 4 ? 4 : vec;
        while (v > 1 && 16 * v >= width) v /= 2;
        const int64_t table = rows * 32 * v * 4, tiles = (width + 32 * v - 1) / (32 * v);
        const int warps = (int)(EMB_TABLE_BYTES / table < EMB_WARPS ? EMB_TABLE_BYTES / table : EMB_WARPS);
        int64_t blocks = grid_max / tiles > 1 ? grid_max / tiles : 1;
        const int64_t least = (tokens + 32 * warps - 1) / (32 * warps);  // 32 tokens a warp at least
        if (blocks > least) blocks = least;
        E.parts = warps;
        E.share = ((tokens + blocks * warps - 1) / (blocks * warps) + 31) / 32 * 32;
        blocks = (tokens + E.share * warps - 1) / (E.share * warps);
        if (tiles < 65536) {
            auto table_kernel = of(v, EMB_TABLE);
            static int configured[64][3][3] = {};
            int dev = 0;
            cudaGetDevice(&dev);
            const int vi = v == 4 ? 2 : v - 1;
            if (dev < 0 || dev >= 64 || !configured[dev][grad_type][vi]) {
                const int rc = cuda_status(cudaFuncSetAttribute(table_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, EMB_TABLE_BYTES),
                                           "embedding_backward: shared memory size");
                if (rc) return rc;
                if (dev >= 0 && dev < 64) configured[dev][grad_type][vi] = 1;
            }
            table_kernel<<<dim3((unsigned)blocks, (unsigned)tiles), 32 * warps, (size_t)(warps * table), s>>>(E);
            const int rc = launch_status("embedding_backward");
            if (rc) return rc;
            embedding_backward_fold_kernel<<<(unsigned)((rows * width + 31) / 32), EMB_THREADS, 0, s>>>(E, (int)blocks);
            return launch_status("embedding_backward: fold");
        }
    }
    EmbNarrow N;
    if (emb_narrow_plan(tokens, rows, width, grid_max, N)) {
        auto narrow = grad_type == EMB_F32 ? emb_narrow_kernel<float>(vec)
                      : grad_type == EMB_BF16 ? emb_narrow_kernel<__nv_bfloat16>(vec) : emb_narrow_kernel<__half>(vec);
        static int configured[64][3][4] = {};
        int dev = 0;
        cudaGetDevice(&dev);
        const int vi = vec == 8 ? 3 : vec == 4 ? 2 : vec - 1;
        if (dev < 0 || dev >= 64 || !configured[dev][grad_type][vi]) {
            const int rc = cuda_status(cudaFuncSetAttribute(narrow, cudaFuncAttributeMaxDynamicSharedMemorySize, EMB_NARROW_SMEM),
                                       "embedding_backward: shared memory size");
            if (rc) return rc;
            if (dev >= 0 && dev < 64) configured[dev][grad_type][vi] = 1;
        }
        narrow<<<dim3((unsigned)N.shares, (unsigned)N.ranges, (unsigned)N.tiles), EMB_THREADS, EMB_NARROW_SMEM, s>>>(E, N);
        const int rc = launch_status("embedding_backward");
        if (rc || N.shares == 1) return rc;
        if (N.shares <= EMB_FOLD_FEW)
            embedding_backward_fold_few_kernel<<<(unsigned)((rows * width + 255) / 256), 256, 0, s>>>(E, (int)N.shares);
        else
            embedding_backward_fold_kernel<<<(unsigned)((rows * width + 31) / 32), EMB_THREADS, 0, s>>>(E, (int)N.shares);
        return launch_status("embedding_backward: fold");
    }
    auto kernel = of(vec, EMB_SORT);
    if (grid == 1) {
        kernel<<<1, EMB_THREADS, 0, s>>>(E);
        return launch_status("embedding_backward");
    }
    int rc = cuda_status(cudaMemsetAsync(E.barrier, 0, 8, s), "embedding_backward: barrier");
    if (rc) return rc;
    void* args[] = {&E};
    return cuda_status(cudaLaunchCooperativeKernel((const void*)kernel, dim3((unsigned)grid), dim3(EMB_THREADS), args, 0, s),
                       "embedding_backward: cooperative launch");
}

}  // extern "C"
