// Rows of a token table times a scale, and the gradient of the table summed over equal tokens, for vocabularies of any size.
//
//   lookup     out[i] = scale * E[id_i], a zero row where id_i lies outside the vocabulary
//   gradient   dE[t]  = scale * sum of g[i] over the rows i with id_i = t
//
// The sums repeat bit for bit, without atomics on floating values: the rows are ordered by token (a stable counting sort of (token, row) pairs,
// 8 bytes a row), pieces of the order are summed by warps, and what a token has in several pieces is added in the order of the pieces.  Up to 512 rows
// need no order: the block of a token's first row looks for the others.
//
// Bound by memory where there are many columns: a gradient reads n rows once and writes the table once.  1.4M rows x 128 float32, 1000 tokens: lookup 108 us in a row of
// lookups (6.6 TB/s written) and 130 between other calls, whose lines it first drives out of the L2; gradient 156 us, single launches by the profiler 30 for the sort, 112
// for the sums (6.4 TB/s read) and 14 for the joins.  65,537 x 1024 bfloat16, 50,021 tokens: 30 and 88 us (134 MB read, 205 written); sort 30, sums 65, joins 7, which
// overlap where each launch is placed early.  Between a thousand and a hundred thousand rows the chain of short launches is what is left: 15 us at 600 x 128, 19 at
// 5000 x 256, 46 at 20,000 x 512 of 50,000 tokens (100 MB written).
// Rows that are no whole 16-byte pieces, or off 16-byte boundaries, go element by element: 2.7M x 65 float32 329 and 976 us where 2.8M x 64 take 107 and 210, 1.4M x 128
// off boundaries 670 (bfloat16: 309 and 1044, 77 and 253, 710).
// Not kept: one cooperative launch with grid barriers for the whole sort (93 us where 90), pairs ordered in shared memory before they
// are written (a pass of 1.4M rows 21 us where 17.5), pieces of eight bytes for narrow rows (52 us where 53 at 300,000 x 64).
#include <cuda_runtime.h>

#include <cstdint>
#include <mutex>
#include <set>
#include <type_traits>
#include <utility>

#include "../../include/agpt_b200.h"
#include "internal.h"
#include "pdl.cuh"
#include "tc100.cuh"
#include "vec.cuh"

namespace {

using bf16 = __nv_bfloat16;

int launch_status(const char *who) {
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return agpt_set_error(AGPT_E_CUDA, "%s: %s", who, cudaGetErrorString(e));
    return AGPT_OK;
}

// the token of row i, or `vocab` where it lies outside the vocabulary
__device__ __forceinline__ uint32_t token_of(const void *ids, int wide, int64_t i, uint32_t vocab) {
    if (wide) {
        const int64_t t = __ldg(reinterpret_cast<const long long *>(ids) + i);
        return t >= 0 && t < (int64_t)vocab ? (uint32_t)t : vocab;
    }
    const uint32_t t = (uint32_t)__ldg(reinterpret_cast<const int *>(ids) + i);
    return t < vocab ? t : vocab;
}

// ---- lookup: a group of 2^lanes_log2 lanes per row, LOOK_ROWS rows of it in flight -------------------------------------------------
constexpr int LOOK_ROWS = 4;
template <typename T, int VEC>
__global__ void __launch_bounds__(256) lookup_kernel(const T *__restrict__ emb, int64_t ld, const void *__restrict__ ids, int wide, T *__restrict__ out,
                                                      int64_t n, int d, uint32_t vocab, float scale, int lanes_log2) {
    pdl_wait();
    pdl_next();
    const int lanes = 1 << lanes_log2, per_block = 256 >> lanes_log2;
    const int c0 = (threadIdx.x & (lanes - 1)) * VEC;
    const int64_t r0 = (int64_t)blockIdx.x * per_block * LOOK_ROWS + (threadIdx.x >> lanes_log2);
    uint32_t id[LOOK_ROWS];
#pragma unroll
    for (int u = 0; u < LOOK_ROWS; u++) {
        const int64_t r = r0 + (int64_t)u * per_block;
        id[u] = r < n ? token_of(ids, wide, r, vocab) : vocab;
    }
    for (int c = c0; c < d; c += lanes * VEC) {
        vec::Piece<T, VEC> piece[LOOK_ROWS];
#pragma unroll
        for (int u = 0; u < LOOK_ROWS; u++) piece[u].fetch_kept(emb + (int64_t)id[u] * ld + c, id[u] < vocab);
#pragma unroll
        for (int u = 0; u < LOOK_ROWS; u++) {
            const int64_t r = r0 + (int64_t)u * per_block;
            if (r >= n) break;
            float v[VEC];
            piece[u].values(v);
            if (id[u] < vocab)                         // zero rows stay zero whatever the scale is
#pragma unroll
                for (int i = 0; i < VEC; i++) v[i] *= scale;
            vec::store_past<VEC>(out + r * d + c, v);
        }
    }
}

// ---- order of the rows by token: counting sort, least significant digit first -----------------------------------------------------
// A pass counts the digits of each block's rows (count_kernel), turns the counts into places over the blocks (place_kernel) and moves
// the pairs (move_kernel): a warp of a block owns a run of rows and has its own counters, so rows of one digit keep their order.
constexpr int MOVE_WARPS = 16, DIGIT_BITS_MAX = 11, PLACE_RUNS = 32;

// What a pass reads: the caller's tokens, int32 or int64, or the pairs of the pass before.  Known to the compiler, and loads are made without a branch around
// them (behind the last row the last one again): a loop of guarded loads waits for each in turn (the counts of 1.4M rows took 13 us).
enum { IDS32, IDS64, PAIRS };
template <int SOURCE> __device__ __forceinline__ uint32_t key_at(const void *source, int64_t i, uint32_t vocab) {
    if constexpr (SOURCE == PAIRS) return __ldg(&reinterpret_cast<const uint2 *>(source)[i].x);
    else return token_of(source, SOURCE == IDS64, i, vocab);
}
template <int SOURCE> __device__ __forceinline__ uint2 pair_at(const void *source, int64_t i, uint32_t vocab) {
    if constexpr (SOURCE == PAIRS) return __ldg(reinterpret_cast<const uint2 *>(source) + i);
    else return make_uint2(token_of(source, SOURCE == IDS64, i, vocab), (uint32_t)i);
}

template <int SOURCE>
__global__ void __launch_bounds__(256) count_kernel(const void *__restrict__ source, int64_t n, int64_t chunk, uint32_t vocab, int shift, int bins,
                                                     uint32_t *__restrict__ counts) {
    pdl_wait();
    pdl_next();
    extern __shared__ uint32_t s_hist[];
    for (int b = threadIdx.x; b < bins; b += 256) s_hist[b] = 0;
    __syncthreads();
    const int64_t i0 = (int64_t)blockIdx.x * chunk, i1 = min(i0 + chunk, n);
    for (int64_t i = i0 + threadIdx.x; i < i1; i += 256 * 8) {
        uint32_t key[8];
#pragma unroll
        for (int k = 0; k < 8; k++) key[k] = key_at<SOURCE>(source, min(i + 256 * k, i1 - 1), vocab);
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (i + 256 * k < i1) atomicAdd(&s_hist[(key[k] >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += 256) counts[(int64_t)blockIdx.x * bins + b] = s_hist[b];
}

// counts[block][digit] -> rows of the digit in earlier blocks; totals[digit].  A block has 32 digits and PLACE_RUNS runs of the blocks.
__global__ void __launch_bounds__(PLACE_RUNS * 32) place_kernel(uint32_t *__restrict__ counts, int blocks, int bins, uint32_t *__restrict__ totals) {
    pdl_wait();
    pdl_next();
    __shared__ uint32_t s[PLACE_RUNS][32];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, d = blockIdx.x * 32 + lane;
    const int b0 = blocks * w / PLACE_RUNS, b1 = blocks * (w + 1) / PLACE_RUNS;
    uint32_t sum = 0;
    if (d < bins)
#pragma unroll 8
        for (int b = b0; b < b1; b++) sum += counts[(int64_t)b * bins + d];
    s[w][lane] = sum;
    __syncthreads();
    uint32_t at = 0;
    for (int k = 0; k < w; k++) at += s[k][lane];
    if (d >= bins) return;
    if (w == PLACE_RUNS - 1) totals[d] = at + sum;
    for (int first = b0; first < b1; first += 8) {
        uint32_t x[8];
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = first + k < b1 ? counts[(int64_t)(first + k) * bins + d] : 0;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            if (first + k >= b1) break;
            counts[(int64_t)(first + k) * bins + d] = at;
            at += x[k];
        }
    }
}

template <int SOURCE>
__global__ void __launch_bounds__(MOVE_WARPS * 32) move_kernel(const void *__restrict__ source, int64_t n, int64_t chunk, uint32_t vocab, int shift, int bits, const uint32_t *__restrict__ counts,
                                                                const uint32_t *__restrict__ totals, uint2 *__restrict__ out) {
    pdl_wait();
    pdl_next();
    extern __shared__ uint32_t s_at[];                     // [MOVE_WARPS][bins] counters, then places; [bins] starts of the digits
    const int bins = 1 << bits, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    uint32_t *mine = s_at + w * bins, *start = s_at + MOVE_WARPS * bins;
    __shared__ uint32_t s_warp[MOVE_WARPS];
    for (int b = threadIdx.x; b < MOVE_WARPS * bins; b += MOVE_WARPS * 32) s_at[b] = 0;
    // starts of the digits: a thread has neighbours, or none
    const int each = (bins + MOVE_WARPS * 32 - 1) / (MOVE_WARPS * 32);
    uint32_t sum = 0;
    for (int k = 0; k < each; k++) {
        const int b = threadIdx.x * each + k;
        if (b < bins) sum += __ldg(totals + b);
    }
    uint32_t run = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += x;
    }
    if (lane == 31) s_warp[w] = run;
    __syncthreads();
    uint32_t at = run - sum;
    for (int k = 0; k < w; k++) at += s_warp[k];
    for (int k = 0; k < each; k++) {
        const int b = threadIdx.x * each + k;
        if (b < bins) { start[b] = at; at += __ldg(totals + b); }
    }
    // digits of each warp's rows
    const int64_t own = chunk / MOVE_WARPS, i0 = (int64_t)blockIdx.x * chunk + w * own, i1 = min(i0 + own, n);
    for (int64_t i = i0 + lane; i < i1; i += 32 * 8) {
        uint32_t key[8];
#pragma unroll
        for (int k = 0; k < 8; k++) key[k] = key_at<SOURCE>(source, min(i + 32 * k, i1 - 1), vocab);
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (i + 32 * k < i1) atomicAdd(&mine[(key[k] >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += MOVE_WARPS * 32) {
        uint32_t t = start[b] + __ldg(counts + (int64_t)blockIdx.x * bins + b);
#pragma unroll
        for (int k = 0; k < MOVE_WARPS; k++) {
            const uint32_t x = s_at[k * bins + b];
            s_at[k * bins + b] = t;
            t += x;
        }
    }
    __syncthreads();
    if (i0 >= i1) return;
    const auto load = [&](int64_t i) { return pair_at<SOURCE>(source, min(i, i1 - 1), vocab); };
    uint2 next = load(i0 + lane);
    for (int64_t i = i0; i < i1; i += 32) {
        const bool live = i + lane < i1;
        const uint2 p = next;
        next = load(i + 32 + lane);
        const uint32_t digit = live ? (p.x >> shift) & (bins - 1) : 0xffffffffu;
        const uint32_t same = __match_any_sync(0xffffffffu, digit);
        uint32_t to = 0;
        if (live) to = mine[digit] + __popc(same & ((1u << lane) - 1));
        __syncwarp();
        if (live) {
            if (lane == 31 - __clz(same)) mine[digit] = to + 1;      // the last of them
            out[to] = p;
        }
        __syncwarp();
    }
}

// ---- the same in one cluster: up to CLUSTER_ROWS rows -----------------------------------------------------------------------------
// Eight blocks hold all pairs in shared memory and exchange counts and pairs there, digits of eight bits a pass.  Three launches a pass of a few microseconds each are
// most of a gradient of so few rows (whole gradients, one cluster and launches per pass, us):
//   tokens x columns           4096 rows       16,384        24,576        32,768        45,000        65,536
//   200 x 64      (1 / 1 pass) 13.1 / 16.0   15.6 / 18.7   17.8 / 20.6   19.4 / 21.8   22.0 / 22.9   27.3 / 27.3
//   1400 x 128    (2 / 1)      16.1 / 18.5   19.5 / 20.4   22.2 / 21.0   23.6 / 23.1   27.4 / 23.7   36.0 / 28.1
//   50,000 x 256  (2 / 2)      24.0 / 31.0   27.6 / 34.3   30.7 / 36.7   34.2 / 38.8   41.4 / 42.7   50.1 / 49.2
// So the limit is where the middle row has turned and the others have not; twice the rows would fit in shared memory, but eight SMs then take longer than all of them.
constexpr int CLUSTER = 8, CLUSTER_WARPS = 32, CLUSTER_THREADS = CLUSTER_WARPS * 32, CLUSTER_BITS = 8, CLUSTER_BINS = 1 << CLUSTER_BITS;
constexpr int CLUSTER_CHUNK = 4 * 1024, CLUSTER_ROWS = CLUSTER * CLUSTER_CHUNK;
constexpr int CLUSTER_SMEM = 2 * CLUSTER_CHUNK * 8 + (CLUSTER_WARPS + 3) * CLUSTER_BINS * 4;

template <int SOURCE>
__global__ void __launch_bounds__(CLUSTER_THREADS) cluster_sort_kernel(const void *__restrict__ source, int n, int chunk, uint32_t vocab, int passes, uint2 *__restrict__ out) {
    pdl_wait();
    pdl_next();
    extern __shared__ __align__(16) uint32_t s_sort[];
    uint2 *const pairs = reinterpret_cast<uint2 *>(s_sort);                        // [2][chunk]
    uint32_t *const s_at = s_sort + 4 * chunk;                                     // counters, then places, of each warp [CLUSTER_WARPS][bins]
    uint32_t *const s_total = s_at + CLUSTER_WARPS * CLUSTER_BINS, *const s_before = s_total + 2 * CLUSTER_BINS;      // digits of this block, by pass parity; of earlier blocks
    __shared__ uint32_t s_warp[CLUSTER_WARPS];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, rank = blockIdx.x, own = chunk / CLUSTER_WARPS;
    const int first = rank * chunk, rows = max(0, min(chunk, n - first)), i0 = w * own, i1 = min(i0 + own, rows);     // places of this block, and of this warp in it
    uint32_t *const mine = s_at + w * CLUSTER_BINS;
    // The first pass reads the tokens, the others the pairs in shared memory (known to the compiler: see above)
    const auto one_pass = [&](auto from, int pass) {
        constexpr bool TOKENS = decltype(from)::value;
        const int shift = pass * CLUSTER_BITS;
        const uint2 *const in = pairs + (pass & 1 ? 0 : chunk);                    // pass p writes half p & 1
        const uint32_t into = tc::smem_u32(pairs + (pass & 1 ? chunk : 0));
        const auto load = [&](int i) {
            if constexpr (TOKENS) return pair_at<SOURCE>(source, first + i, vocab);
            else return in[i];
        };
        for (int b = threadIdx.x; b < CLUSTER_WARPS * CLUSTER_BINS; b += CLUSTER_THREADS) s_at[b] = 0;
        __syncthreads();
        for (int i = i0 + lane; i < i1; i += 32 * 4) {
            uint32_t key[4];
#pragma unroll
            for (int k = 0; k < 4; k++) key[k] = load(min(i + 32 * k, i1 - 1)).x;
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (i + 32 * k < i1) atomicAdd(&mine[(key[k] >> shift) & (CLUSTER_BINS - 1)], 1u);
        }
        __syncthreads();
        // a thread has a digit: its pairs in the warps before, its total here; then, with the other blocks' totals, its start
        uint32_t *const total = s_total + (pass & 1) * CLUSTER_BINS;
        if (threadIdx.x < CLUSTER_BINS) {
            uint32_t at = 0;
#pragma unroll 8
            for (int k = 0; k < CLUSTER_WARPS; k++) {
                const uint32_t x = s_at[k * CLUSTER_BINS + threadIdx.x];
                s_at[k * CLUSTER_BINS + threadIdx.x] = at;
                at += x;
            }
            total[threadIdx.x] = at;
        }
        tc::cluster_sync();                            // totals are there; every block has read the half that this pass writes
        uint32_t all = 0, before = 0;
        if (threadIdx.x < CLUSTER_BINS) {
            const uint32_t here = tc::smem_u32(total + threadIdx.x);
            uint32_t x[CLUSTER];
#pragma unroll
            for (int r = 0; r < CLUSTER; r++) x[r] = tc::peer_lds_u1(tc::peer_addr(here, r));
#pragma unroll
            for (int r = 0; r < CLUSTER; r++) {
                all += x[r];
                if (r < rank) before += x[r];
            }
        }
        uint32_t run = all;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += x;
        }
        if (lane == 31) s_warp[w] = run;
        __syncthreads();
        if (threadIdx.x < CLUSTER_BINS) {
            uint32_t at = run - all + before;
            for (int k = 0; k < w; k++) at += s_warp[k];
            s_before[threadIdx.x] = at;
        }
        __syncthreads();
        for (int i = i0; i < i1; i += 32 * 4) {
            uint2 p[4];
#pragma unroll
            for (int r = 0; r < 4; r++) p[r] = load(min(i + 32 * r + lane, i1 - 1));
#pragma unroll
            for (int r = 0; r < 4; r++) {
                if (i + 32 * r >= i1) break;
                const bool live = i + 32 * r + lane < i1;
                const uint32_t digit = (p[r].x >> shift) & (CLUSTER_BINS - 1);
                uint32_t same = __ballot_sync(0xffffffffu, live);
#pragma unroll
                for (int k = 0; k < CLUSTER_BITS; k++) {
                    const bool one = digit >> k & 1;
                    const uint32_t ones = __ballot_sync(0xffffffffu, one);
                    same &= one ? ones : ~ones;
                }
                uint32_t at = 0;
                if (live) at = mine[digit] + __popc(same & ((1u << lane) - 1));
                __syncwarp();
                if (live) {
                    if (lane == 31 - __clz(same)) mine[digit] = at + 1;      // the last of them
                    const uint32_t to = s_before[digit] + at;
                    if (pass + 1 == passes) out[to] = p[r];
                    else {
                        const uint32_t block = to / (uint32_t)chunk;
                        tc::peer_sts_u2(tc::peer_addr(into + (to - block * chunk) * 8, block), p[r].x, p[r].y);
                    }
                }
                __syncwarp();
            }
        }
        if (pass + 1 < passes) tc::cluster_sync();     // pairs are there
    };
    one_pass(std::true_type(), 0);
    for (int pass = 1; pass < passes; pass++) one_pass(std::false_type(), pass);
    tc::cluster_sync();                                // no block leaves while another may read its totals
}

// ---- sums over the ordered rows ----------------------------------------------------------------------------------------------------
// A warp has `run` places of the order (64, fewer while there are less than eight blocks an SM) and 32 * VEC columns, a block SUM_WARPS warps side by side.  Tokens that end where they began are
// written; the warps' first and last sums meet in shared memory; what a block has of a token that began before it goes to head[block], of
// one that goes on behind it to tail[block], and join_kernel adds tail and heads in order.
constexpr int SUM_WARPS = 8, SUM_RING = 8, FILL_TOKENS = 64;

template <typename O, int VEC>
__device__ __forceinline__ void write_row(O *out, int64_t at, float (&v)[VEC], float scale, int accumulate) {
    if (accumulate) {
        float old[VEC];
#pragma unroll
        for (int i = 0; i < VEC; i++) old[i] = (float)out[at + i];
#pragma unroll
        for (int i = 0; i < VEC; i++) v[i] = old[i] + scale * v[i];
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i++) v[i] *= scale;
    }
    vec::store_past<VEC>(out + at, v);
}

// zero rows of the tokens that no row has
template <typename O>
__device__ void fill_absent(const uint2 *order, int64_t n, O *out, int d, uint32_t vocab, int64_t first) {
    __shared__ uint32_t s_absent[FILL_TOKENS / 32];
    if (threadIdx.x < FILL_TOKENS) {
        const int64_t t = first + threadIdx.x;
        bool absent = false;
        if (t < vocab) {
            int64_t lo = 0, hi = n;
            while (lo < hi) {
                const int64_t mid = (lo + hi) >> 1;
                if (__ldg(&order[mid].x) < (uint32_t)t) lo = mid + 1; else hi = mid;
            }
            absent = lo >= n || __ldg(&order[lo].x) != (uint32_t)t;
        }
        const uint32_t b = __ballot_sync(0xffffffffu, absent);
        if ((threadIdx.x & 31) == 0) s_absent[threadIdx.x >> 5] = b;
    }
    __syncthreads();
    const bool wide = (d * sizeof(O)) % 16 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
    for (int k = threadIdx.x >> 5; k < FILL_TOKENS; k += blockDim.x >> 5) {
        if (!(s_absent[k >> 5] >> (k & 31) & 1)) continue;
        O *row = out + (first + k) * (int64_t)d;
        if (wide)
            for (int c = threadIdx.x & 31; c < (int)(d * sizeof(O) / 16); c += 32) reinterpret_cast<uint4 *>(row)[c] = make_uint4(0, 0, 0, 0);
        else
            for (int c = threadIdx.x & 31; c < d; c += 32) row[c] = (O)0.f;
    }
}

template <typename T, typename O, int VEC>
__global__ void __launch_bounds__(SUM_WARPS * 32, 4) sum_kernel(const T *__restrict__ grad, int64_t ld, const uint2 *__restrict__ order, int64_t n, int d, uint32_t vocab,
                                                              int run, int64_t blocks, float scale, int accumulate, O *__restrict__ out, float *__restrict__ head,
                                                              float *__restrict__ tail) {
    pdl_wait();
    pdl_next();
    constexpr int COLS = 32 * VEC;
    extern __shared__ __align__(16) unsigned char s_rows[];     // VEC > 1: [SUM_WARPS][SUM_RING] rows of 512 bytes
    __shared__ float s_part[SUM_WARPS][2][COLS];
    __shared__ uint32_t s_first[SUM_WARPS], s_last[SUM_WARPS];
    __shared__ uint8_t s_in[SUM_WARPS], s_out[SUM_WARPS], s_through[SUM_WARPS];
    if (blockIdx.x >= blocks) {
        if (blockIdx.y == 0) fill_absent(order, n, out, d, vocab, (blockIdx.x - blocks) * FILL_TOKENS);
        return;
    }
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.y * COLS + lane * VEC;
    const int64_t p0 = ((int64_t)blockIdx.x * SUM_WARPS + w) * run, p1 = min(p0 + run, n);
    if (p0 < n) {
        const uint2 near = __ldg(order + min(p0 + lane, p1 - 1)), far = __ldg(order + min(p0 + 32 + lane, p1 - 1));      // at most 64 places
        float acc[VEC];
#pragma unroll
        for (int i = 0; i < VEC; i++) acc[i] = 0.f;
        const uint32_t first = __ldg(&order[p0].x), last = __ldg(&order[p1 - 1].x), ahead = __ldg(&order[max(p0 - 1, (int64_t)0)].x), behind = __ldg(&order[min(p1, n - 1)].x);
        const bool in = p0 > 0 && ahead == first, goes_on = p1 < n && behind == last;
        uint32_t cur = first;
        bool begun_before = in;
        // rows outside the vocabulary are last: a warp that begins with one has nothing to add, and sums of theirs are written nowhere
        const int live = first < vocab ? (int)(p1 - p0) : 0;
        // bit k: place k has another token than place k - 1
        const uint32_t left = __shfl_up_sync(0xffffffffu, near.x, 1), left2 = __shfl_up_sync(0xffffffffu, far.x, 1), middle = __shfl_sync(0xffffffffu, near.x, 31);
        const uint64_t change = (uint64_t)__ballot_sync(0xffffffffu, far.x != (lane ? left2 : middle)) << 32 | __ballot_sync(0xffffffffu, lane && near.x != left);
        const auto row_at = [&](int k) { return __shfl_sync(0xffffffffu, k < 32 ? near.y : far.y, k & 31); };
        const auto next_token = [&](int k) {
            if (begun_before) {
#pragma unroll
                for (int i = 0; i < VEC; i++) s_part[w][0][lane * VEC + i] = acc[i];
            } else if (cur < vocab && c < d) write_row<O, VEC>(out, (int64_t)cur * d + c, acc, scale, accumulate);
            cur = __shfl_sync(0xffffffffu, k < 32 ? near.x : far.x, k & 31);
            begun_before = false;
#pragma unroll
            for (int i = 0; i < VEC; i++) acc[i] = 0.f;
        };
        if constexpr (VEC > 1) {
            // Rows come by asynchronous copies into a ring that only the copying lane reads: SUM_RING rows of every warp are on their way without a register each.
            // (Eight rows in registers at a time left the loads waiting for the sums: 142 us of this kernel at 1.4M x 128, two batches of four 150 and more, this 113.)
            const uint32_t ring = (uint32_t)__cvta_generic_to_shared(s_rows) + (w * SUM_RING * 32 + lane) * 16;
            const auto fetch = [&](int k) {
                if (k < live) {
                    const T *from = grad + (int64_t)row_at(k) * ld + c;
                    if (c < d) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ring + (k % SUM_RING) * 512), "l"(from) : "memory");
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
#pragma unroll
            for (int k = 0; k < SUM_RING - 1; k++) fetch(k);
            for (int k0 = 0; k0 < live; k0 += SUM_RING)
#pragma unroll
                for (int u = 0; u < SUM_RING; u++) {
                    const int k = k0 + u;
                    if (k >= live) break;
                    fetch(k + SUM_RING - 1);
                    asm volatile("cp.async.wait_group %0;" ::"n"(SUM_RING - 1) : "memory");
                    vec::Piece<T, VEC> piece;
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(piece.w[0]), "=r"(piece.w[1]), "=r"(piece.w[2]), "=r"(piece.w[3]) : "r"(ring + u * 512) : "memory");
                    float v[VEC];
                    piece.values(v);
                    if (change >> k & 1) next_token(k);
#pragma unroll
                    for (int i = 0; i < VEC; i++) acc[i] += v[i];
                }
        } else {
            constexpr int U = 8;
            for (int k0 = 0; k0 < live; k0 += U) {
                vec::Piece<T, VEC> piece[U];
#pragma unroll
                for (int u = 0; u < U; u++) piece[u].fetch(grad + (int64_t)row_at(k0 + u) * ld + c, k0 + u < live && c < d);
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (k0 + u >= live) break;
                    float v[VEC];
                    piece[u].values(v);
                    if (change >> (k0 + u) & 1) next_token(k0 + u);
#pragma unroll
                    for (int i = 0; i < VEC; i++) acc[i] += v[i];
                }
            }
        }
        if (begun_before || goes_on) {
#pragma unroll
            for (int i = 0; i < VEC; i++) s_part[w][begun_before ? 0 : 1][lane * VEC + i] = acc[i];
        } else if (cur < vocab && c < d) write_row<O, VEC>(out, (int64_t)cur * d + c, acc, scale, accumulate);
        if (lane == 0) {
            s_first[w] = first; s_last[w] = last;
            s_in[w] = in; s_out[w] = goes_on; s_through[w] = begun_before && goes_on;
        }
    }
    __syncthreads();
    // the warps in order; a thread has a column
    const int64_t b0 = (int64_t)blockIdx.x * SUM_WARPS * run;
    const int warps = (int)min((int64_t)SUM_WARPS, (n - b0 + run - 1) / run);
    for (int k = threadIdx.x; k < COLS; k += SUM_WARPS * 32) {
        const int col = blockIdx.y * COLS + k;
        if (col >= d) break;
        float acc = 0.f;
        bool open = false, before = false;
        for (int i = 0; i < warps; i++) {
            if (s_in[i]) {
                if (!open) { open = before = true; acc = 0.f; }           // the block before had its beginning
                acc += s_part[i][0][k];
                if (s_through[i]) continue;
                if (before) head[(int64_t)blockIdx.x * d + col] = acc;
                else if (s_first[i] < vocab) {
                    float one[1] = {acc};
                    write_row<O, 1>(out, (int64_t)s_first[i] * d + col, one, scale, accumulate);
                }
                open = false;
            }
            if (s_out[i]) { open = true; before = false; acc = s_part[i][1][k]; }
        }
        if (open) (before ? head : tail)[(int64_t)blockIdx.x * d + col] = acc;
    }
}

// Tokens that began in a block of the sums and go on behind it: tail, then the heads of the blocks that begin with the token.  A warp has a block; where the heads
// are many, all warps of the block come together and have a run of them each: from 17 on, 157 us at 1.4M x 128 of 1000 tokens and 168 of three; from 5 on 162 and 195, from 65
// on 157 and 168 (25.2 where 23.8 at 40,000 x 256 of 40 tokens).
constexpr int JOIN_ALONE = 16;
template <typename O>
__global__ void __launch_bounds__(256) join_kernel(const uint2 *__restrict__ order, int64_t n, int d, uint32_t vocab, int64_t span, int64_t blocks, float scale, int accumulate,
                                                    O *__restrict__ out, const float *__restrict__ head, const float *__restrict__ tail) {
    pdl_wait();
    pdl_next();
    __shared__ float s_part[8][128];
    __shared__ int64_t s_heads[8];
    __shared__ uint32_t s_key[8];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c0 = blockIdx.y * 128;
    const bool whole = (d & 3) == 0;
    // sums of heads [h0, h1) behind block b, and of its tail; four columns a lane, neighbours if they lie on 16-byte boundaries
    const auto column = [&](int i) { return c0 + (whole ? lane * 4 + i : lane + 32 * i); };
    const auto add = [&](int64_t b, int64_t h0, int64_t h1, bool with_tail, float (&acc)[4]) {
#pragma unroll
        for (int i = 0; i < 4; i++) acc[i] = with_tail && column(i) < d ? tail[b * d + column(i)] : 0.f;
        if (whole) {
            if (column(0) < d)
#pragma unroll 8
                for (int64_t h = h0; h < h1; h++) {
                    const float4 v = __ldcs(reinterpret_cast<const float4 *>(head + (b + 1 + h) * d + column(0)));
                    acc[0] += v.x; acc[1] += v.y; acc[2] += v.z; acc[3] += v.w;
                }
        } else {
#pragma unroll 2
            for (int64_t h = h0; h < h1; h++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (column(i) < d) acc[i] += __ldcs(head + (b + 1 + h) * d + column(i));
        }
    };
    const int64_t b = (int64_t)blockIdx.x * 8 + w, p0 = b * span, p1 = p0 + span;
    int64_t heads = 0;
    uint32_t key = vocab;
    if (b < blocks && p1 < n) {
        // four loads at once
        key = __ldg(&order[p1 - 1].x);
        const uint32_t behind = __ldg(&order[p1].x), first = __ldg(&order[p0].x), ahead = __ldg(&order[max(p0 - 1, (int64_t)0)].x);
        const bool goes_on = key < vocab && behind == key, before = p0 > 0 && first == key && ahead == key;
        if (goes_on && !before) {
            // blocks behind that begin with the token: they are the first ones, so 32 are asked at a time, near ones first, then by 32nds of what is left
            int64_t low = 1, high = blocks - b;                        // `low` of them are known to, from `high` on none does
            for (int64_t step = 1; low < high; step = (high - low + 31) / 32) {
                const int64_t h = low + lane * step, p = p1 + h * span;
                const int yes = __popc(__ballot_sync(0xffffffffu, h < high && p < n && __ldg(&order[p].x) == key));
                if (yes < 32) high = min(high, low + yes * step);
                low = yes ? low + (yes - 1) * step + 1 : low;
                if (yes == 0) break;
            }
            heads = low;
        }
    }
    if (heads && heads <= JOIN_ALONE) {
        float acc[4];
        add(b, 0, heads, true, acc);
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (column(i) < d) {
                float one[1] = {acc[i]};
                write_row<O, 1>(out, (int64_t)key * d + column(i), one, scale, accumulate);
            }
    }
    if (lane == 0) { s_heads[w] = heads; s_key[w] = key; }
    __syncthreads();
    for (int k = 0; k < 8; k++) {
        const int64_t many = s_heads[k];
        if (many <= JOIN_ALONE) continue;
        float acc[4];
        add((int64_t)blockIdx.x * 8 + k, many * w / 8, many * (w + 1) / 8, w == 0, acc);
#pragma unroll
        for (int i = 0; i < 4; i++) s_part[w][lane + 32 * i] = acc[i];
        __syncthreads();
        if (w == 0)
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (column(i) < d) {
                    float one[1] = {0.f};
                    for (int x = 0; x < 8; x++) one[0] += s_part[x][lane + 32 * i];
                    write_row<O, 1>(out, (int64_t)s_key[k] * d + column(i), one, scale, accumulate);
                }
        __syncthreads();
    }
}

// ---- few rows: one launch, no order -------------------------------------------------------------------------------------------------
// Every block reads all tokens; the block of a token's first row adds its rows, a run of the rows per warp; blocks behind fill absent tokens.
// Every block looks at all rows, so the work grows with their square, but up to the limit it is far below what the order costs (here / by the cluster, us): 256 rows x 384, 1400 tokens
// 3.9 / 12.7, 512 4.7 / 13.1; 512 x 128 of 65 tokens 3.5 / 10.2.  1024 rows would still be ahead: 7.4 / 14.2 and 5.5 / 11.5.
constexpr int FEW_ROWS = 512;
template <typename T, typename O, int VEC>
__global__ void __launch_bounds__(256) few_rows_kernel(const T *__restrict__ grad, int64_t ld, const void *__restrict__ ids, int wide, int n, int d, uint32_t vocab,
                                                        float scale, int accumulate, O *__restrict__ out) {
    pdl_wait();
    pdl_next();
    constexpr int COLS = 32 * VEC;
    __shared__ uint32_t s_id[FEW_ROWS];
    __shared__ float s_part[8][COLS];
    __shared__ uint32_t s_present[FILL_TOKENS / 32];
    for (int i = threadIdx.x; i < n; i += 256) s_id[i] = token_of(ids, wide, i, vocab);
    if (threadIdx.x < FILL_TOKENS / 32) s_present[threadIdx.x] = 0;
    __syncthreads();
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    if ((int)blockIdx.x >= n) {
        const int64_t first = (int64_t)(blockIdx.x - n) * FILL_TOKENS;
        if (blockIdx.y) return;
        for (int i = threadIdx.x; i < n; i += 256) {
            const int64_t k = (int64_t)s_id[i] - first;
            if (k >= 0 && k < FILL_TOKENS) atomicOr(&s_present[k >> 5], 1u << (k & 31));
        }
        __syncthreads();
        for (int k = w; k < FILL_TOKENS && first + k < vocab; k += 8) {
            if (s_present[k >> 5] >> (k & 31) & 1) continue;
            for (int c = lane; c < d; c += 32) out[(first + k) * d + c] = (O)0.f;
        }
        return;
    }
    const int self = blockIdx.x;
    const uint32_t id = s_id[self];
    if (id >= vocab) return;
    int earlier = 0;
    for (int i = threadIdx.x; i < self; i += 256) earlier |= s_id[i] == id;
    if (__syncthreads_or(earlier)) return;
    const int c = blockIdx.y * COLS + lane * VEC, left = n - self;
    const int i0 = self + left * w / 8, i1 = self + left * (w + 1) / 8;
    float acc[VEC];
#pragma unroll
    for (int k = 0; k < VEC; k++) acc[k] = 0.f;
    for (int i = i0; i < i1; i += 32) {
        uint32_t hit = __ballot_sync(0xffffffffu, i + lane < i1 && s_id[i + lane] == id);
        while (hit) {
            float v[4][VEC];
            bool have[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                have[u] = hit != 0;
                if (have[u] && c < d) vec::load<VEC>(grad + (int64_t)(i + __ffs(hit) - 1) * ld + c, v[u]);
                hit &= hit - 1;
            }
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (have[u] && c < d)
#pragma unroll
                    for (int k = 0; k < VEC; k++) acc[k] += v[u][k];
        }
    }
#pragma unroll
    for (int k = 0; k < VEC; k++) s_part[w][lane * VEC + k] = acc[k];
    __syncthreads();
    for (int k = threadIdx.x; k < COLS; k += 256) {
        const int col = blockIdx.y * COLS + k;
        if (col >= d) break;
        float one[1] = {0.f};
        for (int i = 0; i < 8; i++) one[0] += s_part[i][k];
        write_row<O, 1>(out, (int64_t)id * d + col, one, scale, accumulate);
    }
}

// ---- sizes ----------------------------------------------------------------------------------------------------------------------------
struct Sizes {
    int passes, bits;              // of the sort; digits of `bits`
    int64_t chunk, chunks;         // rows of a block of the sort
    int run;                       // places of a warp of the sums
    int64_t blocks;                // of the sums
    int64_t at_pairs, at_counts, at_totals, at_head, at_tail, bytes;
};
Sizes sizes_of(int64_t n, int d, int64_t vocab) {
    Sizes z;
    int bits = 0;
    while ((vocab >> bits) > 0) bits++;                       // keys 0 .. vocab
    z.passes = (bits + DIGIT_BITS_MAX - 1) / DIGIT_BITS_MAX;
    z.bits = (bits + z.passes - 1) / z.passes;
    const int64_t sms = vec::sm_count();
    z.chunk = (n + 2 * sms - 1) / (2 * sms);
    z.chunk = z.chunk < 1024 ? 1024 : (z.chunk + 32 * MOVE_WARPS - 1) / (32 * MOVE_WARPS) * (32 * MOVE_WARPS);
    z.chunks = (n + z.chunk - 1) / z.chunk;
    z.run = 64;
    while (z.run > 8 && (n + SUM_WARPS * z.run - 1) / (SUM_WARPS * z.run) * ((d + 127) / 128) < 8 * sms) z.run /= 2;
    z.blocks = (n + SUM_WARPS * z.run - 1) / (SUM_WARPS * z.run);
    const auto up = [](int64_t b) { return (b + 255) / 256 * 256; };
    z.at_pairs = 0;
    z.at_counts = up(n * 8 * (z.passes > 1 ? 2 : 1));
    z.at_totals = z.at_counts + up(z.chunks * (4ll << z.bits));
    z.at_head = z.at_totals + up(4ll << z.bits);
    z.at_tail = z.at_head + up(z.blocks * d * 4);
    z.bytes = z.at_tail + up(z.blocks * d * 4);
    return z;
}

// dynamic shared memory beyond 48 KB, allowed once per kernel and device
template <typename... P>
int allow_smem(void (*kernel)(P...), int bytes) {
    static std::mutex lock;
    static std::set<std::pair<const void *, int>> done;
    int dev = 0;
    cudaGetDevice(&dev);
    std::lock_guard<std::mutex> hold(lock);
    if (done.count({(const void *)kernel, dev})) return AGPT_OK;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return agpt_set_error(AGPT_E_CUDA, "embedding_grad_sorted: %s", cudaGetErrorString(e));
    done.insert({(const void *)kernel, dev});
    return AGPT_OK;
}

template <int SOURCE>
int sort_pass(const void *source, int64_t n, const Sizes &z, uint32_t vocab, int pass, char *ws, uint2 *out, cudaStream_t st) {
    const int bins = 1 << z.bits, shift = pass * z.bits;
    uint32_t *counts = (uint32_t *)(ws + z.at_counts), *totals = (uint32_t *)(ws + z.at_totals);
    const size_t smem = (size_t)(MOVE_WARPS + 1) * bins * 4;
    if (int rc = allow_smem(move_kernel<SOURCE>, (MOVE_WARPS + 1) * 4 << DIGIT_BITS_MAX)) return rc;
    pdl_launch(count_kernel<SOURCE>, (unsigned)z.chunks, 256, (size_t)bins * 4, st, source, n, z.chunk, vocab, shift, bins, counts);
    pdl_launch(place_kernel, (unsigned)((bins + 31) / 32), PLACE_RUNS * 32, 0, st, counts, (int)z.chunks, bins, totals);
    pdl_launch(move_kernel<SOURCE>, (unsigned)z.chunks, MOVE_WARPS * 32, smem, st, source, n, z.chunk, vocab, shift, z.bits, (const uint32_t *)counts,
               (const uint32_t *)totals, out);
    return AGPT_OK;
}

template <int SOURCE>
int sort_in_cluster(const void *ids, int n, uint32_t vocab, uint2 *out, cudaStream_t st) {
    const int own = ((n + CLUSTER * CLUSTER_WARPS - 1) / (CLUSTER * CLUSTER_WARPS) + 31) / 32 * 32, chunk = own * CLUSTER_WARPS;
    int passes = 1;
    while (passes * CLUSTER_BITS < 32 && (vocab >> (passes * CLUSTER_BITS)) > 0) passes++;
    if (int rc = allow_smem(cluster_sort_kernel<SOURCE>, CLUSTER_SMEM)) return rc;
    const size_t smem = (size_t)2 * chunk * 8 + (CLUSTER_WARPS + 3) * CLUSTER_BINS * 4;
    const cudaError_t e = pdl_launch_clusters(cluster_sort_kernel<SOURCE>, CLUSTER, CLUSTER, CLUSTER_THREADS, smem, st, ids, n, chunk, vocab, passes, out);
    if (e != cudaSuccess) return agpt_set_error(AGPT_E_CUDA, "embedding_grad_sorted: %s", cudaGetErrorString(e));
    return AGPT_OK;
}

template <typename T, typename O, int VEC>
int grad_sorted(const T *grad, int64_t ld, const void *ids, int wide, O *out, int64_t n, int d, uint32_t vocab, float scale, int accumulate, char *ws, cudaStream_t st) {
    const unsigned slices = (unsigned)((d + 32 * VEC - 1) / (32 * VEC));
    const int64_t fill = accumulate ? 0 : ((int64_t)vocab + FILL_TOKENS - 1) / FILL_TOKENS;
    if (n <= FEW_ROWS) {
        if (n + fill) pdl_launch(few_rows_kernel<T, O, VEC>, dim3((unsigned)(n + fill), slices), 256, 0, st, grad, ld, ids, wide, (int)n, d, vocab, scale, accumulate, out);
        return launch_status("embedding_grad_sorted");
    }
    const Sizes z = sizes_of(n, d, vocab);
    const uint2 *order;
    if (n <= CLUSTER_ROWS) {
        if (int rc = wide ? sort_in_cluster<IDS64>(ids, (int)n, vocab, (uint2 *)(ws + z.at_pairs), st) : sort_in_cluster<IDS32>(ids, (int)n, vocab, (uint2 *)(ws + z.at_pairs), st)) return rc;
        order = (uint2 *)(ws + z.at_pairs);
    } else {
        uint2 *pairs[2] = {(uint2 *)(ws + z.at_pairs), (uint2 *)(ws + z.at_pairs) + n};
        if (int rc = wide ? sort_pass<IDS64>(ids, n, z, vocab, 0, ws, pairs[0], st) : sort_pass<IDS32>(ids, n, z, vocab, 0, ws, pairs[0], st)) return rc;
        for (int p = 1; p < z.passes; p++)
            if (int rc = sort_pass<PAIRS>(pairs[(p - 1) & 1], n, z, vocab, p, ws, pairs[p & 1], st)) return rc;
        order = pairs[(z.passes - 1) & 1];
    }
    float *head = (float *)(ws + z.at_head), *tail = (float *)(ws + z.at_tail);
    if (VEC > 1)
        if (int rc = allow_smem(sum_kernel<T, O, VEC>, SUM_WARPS * SUM_RING * 512)) return rc;
    pdl_launch(sum_kernel<T, O, VEC>, dim3((unsigned)(z.blocks + fill), slices), SUM_WARPS * 32, VEC > 1 ? SUM_WARPS * SUM_RING * 512 : 0, st, grad, ld, order, n, d, vocab,
               z.run, z.blocks, scale, accumulate, out, head, tail);
    if (z.blocks > 1)
        pdl_launch(join_kernel<O>, dim3((unsigned)((z.blocks + 7) / 8), (unsigned)((d + 127) / 128)), 256, 0, st, order, n, d, vocab, (int64_t)SUM_WARPS * z.run, z.blocks,
                   scale, accumulate, out, (const float *)head, (const float *)tail);
    return launch_status("embedding_grad_sorted");
}

template <typename T>
int lookup(const T *emb, int64_t ld, const void *ids, int wide, T *out, int64_t n, int d, uint32_t vocab, float scale, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    const bool whole = d % V == 0 && ld % V == 0 && vec::aligned(emb, 16) && vec::aligned(out, 16);
    const int pieces = whole ? d / V : d;
    int log2 = 0;
    while (log2 < 5 && (1 << log2) < pieces) log2++;
    const int64_t per_block = (256 >> log2) * LOOK_ROWS;
    const unsigned blocks = (unsigned)((n + per_block - 1) / per_block);
    if (whole) pdl_launch(lookup_kernel<T, V>, blocks, 256, 0, st, emb, ld, ids, wide, out, n, d, vocab, scale, log2);
    else pdl_launch(lookup_kernel<T, 1>, blocks, 256, 0, st, emb, ld, ids, wide, out, n, d, vocab, scale, log2);
    return launch_status("embedding_lookup");
}

template <typename T>
int grad_by_output(const T *grad, int64_t ld, const void *ids, int wide, void *out, int out_type, int64_t n, int d, uint32_t vocab, float scale, int accumulate, char *ws,
                   cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    // whole pieces: both the rows and, written by the same lanes, the table lie on 16-byte boundaries
    const bool whole = d % V == 0 && ld % V == 0 && vec::aligned(grad, 16) && vec::aligned(out, 16);
    const auto run = [&](auto *to) {
        using O = std::remove_pointer_t<decltype(to)>;
        return whole ? grad_sorted<T, O, V>(grad, ld, ids, wide, to, n, d, vocab, scale, accumulate, ws, st)
                     : grad_sorted<T, O, 1>(grad, ld, ids, wide, to, n, d, vocab, scale, accumulate, ws, st);
    };
    return out_type == AGPT_KV_BF16 ? run((bf16 *)out) : run((float *)out);
}

int check_sizes(const char *who, int64_t n, int d, int64_t ld, int64_t vocab, int type) {
    if (n < 0 || d <= 0 || vocab <= 0 || ld < d) return agpt_set_error(AGPT_E_ARG, "%s: bad argument", who);
    if (type != AGPT_KV_F32 && type != AGPT_KV_BF16) return agpt_set_error(AGPT_E_ARG, "%s: rows are float32 (0) or bfloat16 (1)", who);
    if (n > INT32_MAX - 65536 || vocab > INT32_MAX - 65536 || d > 1 << 20) return agpt_set_error(AGPT_E_LIMIT, "%s: more than 2^31 rows or symbols, or 2^20 columns", who);
    return AGPT_OK;
}

}  // namespace

extern "C" int agpt_b200_embedding_lookup(const void *d_emb, int64_t emb_ld, int type, const void *d_ids, int ids64, void *d_out, int64_t n, int d_model, int vocab,
                                          float scale, void *stream) {
    if (int rc = check_sizes("embedding_lookup", n, d_model, emb_ld, vocab, type)) return rc;
    if (n == 0) return AGPT_OK;
    if (!d_emb || !d_ids || !d_out) return agpt_set_error(AGPT_E_ARG, "embedding_lookup: bad argument");
    cudaStream_t st = (cudaStream_t)stream;
    if (type == AGPT_KV_BF16) return lookup((const bf16 *)d_emb, emb_ld, d_ids, ids64, (bf16 *)d_out, n, d_model, (uint32_t)vocab, scale, st);
    return lookup((const float *)d_emb, emb_ld, d_ids, ids64, (float *)d_out, n, d_model, (uint32_t)vocab, scale, st);
}

extern "C" int64_t agpt_b200_embedding_grad_sorted_workspace_bytes(int64_t n, int d_model, int vocab) {
    if (int rc = check_sizes("embedding_grad_sorted_workspace_bytes", n, d_model, d_model, vocab, AGPT_KV_F32)) return rc;
    return n <= FEW_ROWS ? 0 : sizes_of(n, d_model, vocab).bytes;
}

extern "C" int agpt_b200_embedding_grad_sorted(const void *d_grad, int64_t grad_ld, int type, const void *d_ids, int ids64, void *d_emb_grad, int out_type, int64_t n,
                                               int d_model, int vocab, float scale, int accumulate, void *d_workspace, int64_t workspace_bytes, void *stream) try {
    if (int rc = check_sizes("embedding_grad_sorted", n, d_model, grad_ld, vocab, type)) return rc;
    if (out_type != AGPT_KV_F32 && out_type != AGPT_KV_BF16) return agpt_set_error(AGPT_E_ARG, "embedding_grad_sorted: the table's gradient is float32 (0) or bfloat16 (1)");
    if (!d_emb_grad || (n && (!d_grad || !d_ids))) return agpt_set_error(AGPT_E_ARG, "embedding_grad_sorted: bad argument");
    const int64_t need = n <= FEW_ROWS ? 0 : sizes_of(n, d_model, vocab).bytes;
    if (need && (!d_workspace || workspace_bytes < need || !vec::aligned(d_workspace, 16)))
        return agpt_set_error(AGPT_E_ARG, "embedding_grad_sorted: workspace too small (agpt_b200_embedding_grad_sorted_workspace_bytes)");
    cudaStream_t st = (cudaStream_t)stream;
    if (type == AGPT_KV_BF16)
        return grad_by_output((const bf16 *)d_grad, grad_ld, d_ids, ids64, d_emb_grad, out_type, n, d_model, (uint32_t)vocab, scale, accumulate, (char *)d_workspace, st);
    return grad_by_output((const float *)d_grad, grad_ld, d_ids, ids64, d_emb_grad, out_type, n, d_model, (uint32_t)vocab, scale, accumulate, (char *)d_workspace, st);
} AGPT_CATCH("embedding_grad_sorted")
