// RMS norm of queries and keys per head and their rotation by position, in one pass over the rows, forward and backward.
//
//   r = 1 / sqrt(mean(x^2) + eps)   u = r x   y = R(pos) (g u)        for every row and head, g the gain of queries or of keys
//   w = R(pos)^T dy   c = g w       dx = r (c - u mean(c u))          dg += sum over rows and heads of w u
//
// The pairs (2 i, 2 i + 1) of a head turn by the entries 2 i of the tables, as in agpt_b200_rope.  The backward forms r again from x, so the
// forward keeps nothing.  Statistics and sums are float32; bfloat16 rows are rounded once, on the way out.
//
// Bound by memory in float32: 1.4M rows of 4 + 4 heads of 32, forward 427 us (6.7 TB/s), backward 675 (6.4).  In bfloat16 a byte takes twice the arithmetic: 41k rows of
// 32 + 8 heads of 128 167 us (5.0 TB/s, issue slots at 57 %) and 250 (5.0).  A few rows: 2.6 us for 7, 9 for a backward of 1733 with its gain gradients.
// Not kept: two or three heads a group (190 us and more in bfloat16), four columns a bfloat16 lane (202 and 320), four forward blocks an SM (spills, 468 us in
// float32), columns in pairs in the forward as well (482).
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/agpt_b200.h"
#include "internal.h"
#include "pdl.cuh"
#include "tc100.cuh"
#include "vec.cuh"

namespace {

using bf16 = __nv_bfloat16;
using tc::f2;
using tc::f2_add; using tc::f2_fma; using tc::f2_get; using tc::f2_mul; using tc::f2_pack; using tc::f2_same;

// Blocks of the backward on an SM by the bytes of an element of x: in float32 four (674 us at 1.4M x 8 x 32, three 711), in bfloat16, with eight columns a lane, three
constexpr int back_blocks(int bytes) { return bytes == 4 ? 4 : 3; }

struct Rows {                          // queries or keys: heads * head_dim columns, rows ld elements apart
    const void *x, *dy;
    void *out;                         // y, or dx
    int64_t ld_x, ld_dy, ld_out;
    const float *gain;                 // NULL: 1
    int wide_out;                      // out is float32 (else bfloat16)
    int heads, groups;                 // groups of lanes per row
};
struct Heads {
    Rows q, k;
    const int32_t *pos;
    const float *cosv, *sinv;
    int64_t n;
    int hd, n_pos, lanes_log2, groups; // groups of both sides
    float eps, inv_hd;                 // 1 / hd: exact for powers of two, else one rounding
    vec::Divide by_groups;
    float *partial;                    // backward: [blocks][2][hd]
    int64_t tasks;
};

// LOG2 >= 0: the lanes of a group are known to the compiler
template <int LOG2> __device__ __forceinline__ float group_sum(float v, int lanes) {
    if constexpr (LOG2 >= 0) {
#pragma unroll
        for (int o = (1 << LOG2) >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    } else {
        for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    return v;
}
template <int VEC> __device__ __forceinline__ void store_either(void *p, int64_t at, int wide, const float (&v)[VEC]) {
    if (wide) vec::store_past<VEC>(reinterpret_cast<float *>(p) + at, v);
    else vec::store_past<VEC>(reinterpret_cast<bf16 *>(p) + at, v);
}
// VEC entries of a table or a gain, by 16 bytes where the rows allow it
template <int VEC> __device__ __forceinline__ void load_cached(const float *p, float (&v)[VEC]) {
    if constexpr (VEC % 4 == 0) {
#pragma unroll
        for (int i = 0; i < VEC / 4; i++) {
            const float4 x = __ldg(reinterpret_cast<const float4 *>(p) + i);
            v[4 * i] = x.x; v[4 * i + 1] = x.y; v[4 * i + 2] = x.z; v[4 * i + 3] = x.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i++) v[i] = __ldg(p + i);
    }
}
// a piece as pairs of neighbouring columns: two columns an instruction, and the two that turn together
template <typename T, int VEC> __device__ __forceinline__ void pairs(const vec::Piece<T, VEC> &p, f2 (&v)[VEC / 2]) {
    float x[VEC];
    p.values(x);
#pragma unroll
    for (int i = 0; i < VEC / 2; i++) v[i] = f2_pack(x[2 * i], x[2 * i + 1]);
}
template <int VEC> __device__ __forceinline__ void load_gain(const float *gain, int c, float (&v)[VEC]) {
    if (gain) load_cached<VEC>(gain + c, v);
    else
#pragma unroll
        for (int i = 0; i < VEC; i++) v[i] = 1.f;
}

// The reciprocal root is the hardware's (2 ulp at most): next to the sum of squares, whose head_dim / 2 roundings the root leaves, it adds little.
// A group of lanes owns HEADS heads of one side of a row, `groups` of that side apart, so that neighbouring groups read neighbouring heads and the table's
// entries and the gain are read once for HEADS heads; a lane has NV pieces of VEC columns, `lanes` pieces apart.
template <typename T, int VEC, int NV, int HEADS, int LOG2>
__global__ void __launch_bounds__(256) norm_rope_kernel(const __grid_constant__ Heads P) {
    pdl_wait();
    pdl_next();
    const int lanes_log2 = LOG2 >= 0 ? LOG2 : P.lanes_log2, lanes = 1 << lanes_log2, lane = threadIdx.x & (lanes - 1);
    const int64_t task = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> lanes_log2;
    const bool live = task < P.tasks;
    const int64_t row = live ? vec::quotient(task, P.by_groups) : 0;
    int g = (int)(live ? task - row * P.groups : 0);
    const bool is_q = g < P.q.groups;
    const Rows &m = is_q ? P.q : P.k;
    if (!is_q) g -= P.q.groups;
    const int hd = P.hd;
    const T *x = reinterpret_cast<const T *>(m.x) + row * m.ld_x;
    vec::Piece<T, VEC> piece[HEADS][NV];
#pragma unroll
    for (int u = 0; u < HEADS; u++) {
        const int h = g + u * m.groups;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int c = (lane + k * lanes) * VEC;
            piece[u][k].fetch(x + h * hd + c, live && h < m.heads && c < hd);
        }
    }
    // y = r (x0 g0 cos - x1 g1 sin, x0 g0 sin + x1 g1 cos): gain and table are multiplied once for all heads of the group
    float2 from0[NV][VEC / 2], from1[NV][VEC / 2];
    const int at = live ? min(max(__ldg(P.pos + row), 0), P.n_pos - 1) : 0;
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int c = (lane + k * lanes) * VEC;
        if (c >= hd) continue;
        float cs[VEC], sn[VEC], gain[VEC];
        load_cached<VEC>(P.cosv + (int64_t)at * hd + c, cs);
        load_cached<VEC>(P.sinv + (int64_t)at * hd + c, sn);
        load_gain<VEC>(m.gain, c, gain);
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
            from0[k][i / 2] = make_float2(gain[i] * cs[i], gain[i] * sn[i]);
            from1[k][i / 2] = make_float2(-gain[i + 1] * sn[i], gain[i + 1] * cs[i]);
        }
    }
    float r[HEADS], v[HEADS][NV][VEC];
#pragma unroll
    for (int u = 0; u < HEADS; u++) {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            piece[u][k].values(v[u][k]);
#pragma unroll
            for (int i = 0; i < VEC; i++) s += v[u][k][i] * v[u][k][i];
        }
        r[u] = rsqrtf(group_sum<LOG2>(s, lanes) * P.inv_hd + P.eps);
    }
    if (!live) return;
#pragma unroll
    for (int u = 0; u < HEADS; u++) {
        const int h = g + u * m.groups;
        if (h >= m.heads) break;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int c = (lane + k * lanes) * VEC;
            if (c >= hd) break;
            float y[VEC];
#pragma unroll
            for (int i = 0; i < VEC / 2; i++) {
                const float a = v[u][k][2 * i], b = v[u][k][2 * i + 1];
                y[2 * i] = r[u] * (a * from0[k][i].x + b * from1[k][i].x);
                y[2 * i + 1] = r[u] * (a * from0[k][i].y + b * from1[k][i].y);
            }
            store_either<VEC>(m.out, row * m.ld_out + h * hd + c, m.wide_out, y);
        }
    }
}

// The blocks walk the tasks by a multiple of the groups of a row, so that a thread stays with its heads: side, gain and the columns' gain gradients are its own
// for the whole kernel, and the row moves by a constant.  The block adds its groups in order into partial[block].
template <typename T, typename D, int VEC, int NV, int HEADS, int LOG2>
__global__ void __launch_bounds__(256, NV == 1 ? back_blocks(sizeof(T)) : 1) norm_rope_backward_kernel(const __grid_constant__ Heads P, const int64_t row_step) {
    pdl_wait();
    pdl_next();
    extern __shared__ float s_gain[];                  // [groups of the block][2][hd]
    const int lanes_log2 = LOG2 >= 0 ? LOG2 : P.lanes_log2, lanes = 1 << lanes_log2, lane = threadIdx.x & (lanes - 1), per_block = 256 >> lanes_log2,
              own = threadIdx.x >> lanes_log2;
    const int hd = P.hd;
    const int64_t task = (int64_t)blockIdx.x * per_block + own, first = vec::quotient(task, P.by_groups);
    int g = (int)(task - first * P.groups);
    const bool is_q = g < P.q.groups;
    const Rows &m = is_q ? P.q : P.k;
    if (!is_q) g -= P.q.groups;
    f2 sum[NV][VEC / 2], gain[NV][VEC / 2];
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int c = (lane + k * lanes) * VEC;
        float e[VEC];
#pragma unroll
        for (int i = 0; i < VEC; i++) e[i] = 0.f;
        if (c < hd) load_gain<VEC>(m.gain, c, e);
#pragma unroll
        for (int i = 0; i < VEC / 2; i++) { sum[k][i] = 0; gain[k][i] = f2_pack(e[2 * i], e[2 * i + 1]); }
    }
    // A float32 sum over thousands of rows one after the other loses bits: every FLUSH rounds it goes to the thread's own place in shared memory.
    constexpr int FLUSH = 32;
    const auto flush = [&](bool first_time) {
        if (!P.partial) return;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int c = (lane + k * lanes) * VEC;
            if (c < hd)
#pragma unroll
                for (int i = 0; i < VEC; i++) {
                    const float2 t = f2_get(sum[k][i / 2]);
                    float *mine = s_gain + (own * 2 + !is_q) * hd + c + i;
                    *mine = first_time ? 0.f : *mine + (i & 1 ? t.y : t.x);
                    if (first_time) s_gain[(own * 2 + is_q) * hd + c + i] = 0.f;
                }
#pragma unroll
            for (int i = 0; i < VEC / 2; i++) sum[k][i] = 0;
        }
    };
    flush(true);
    const int64_t rounds = (P.n + row_step - 1) / row_step;
    int next = first < P.n ? __ldg(P.pos + first) : 0;     // the table waits for the position: asked for a round ahead
    for (int64_t t = 0; t < rounds; t++) {
        const int64_t row = first + t * row_step;
        const bool live = row < P.n;
        const int at = min(max(next, 0), P.n_pos - 1);
        next = row + row_step < P.n ? __ldg(P.pos + row + row_step) : 0;
        vec::Piece<T, VEC> x_piece[HEADS][NV];
        vec::Piece<D, VEC> d_piece[HEADS][NV];
        const T *at_x = reinterpret_cast<const T *>(m.x) + row * m.ld_x;
        const D *at_d = reinterpret_cast<const D *>(m.dy) + row * m.ld_dy;
#pragma unroll
        for (int u = 0; u < HEADS; u++) {
            const int h = g + u * m.groups;
#pragma unroll
            for (int k = 0; k < NV; k++) {
                const int c = (lane + k * lanes) * VEC;
                x_piece[u][k].fetch(at_x + h * hd + c, live && h < m.heads && c < hd);
                d_piece[u][k].fetch(at_d + h * hd + c, live && h < m.heads && c < hd);
            }
        }
        float cs[NV][VEC / 2], sn[NV][VEC / 2];
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int c = (lane + k * lanes) * VEC;
#pragma unroll
            for (int i = 0; i < VEC / 2; i++) cs[k][i] = sn[k][i] = 0.f;
            if (c >= hd) continue;
            float e[VEC];
            load_cached<VEC>(P.cosv + (int64_t)at * hd + c, e);
#pragma unroll
            for (int i = 0; i < VEC / 2; i++) cs[k][i] = e[2 * i];
            load_cached<VEC>(P.sinv + (int64_t)at * hd + c, e);
#pragma unroll
            for (int i = 0; i < VEC / 2; i++) sn[k][i] = e[2 * i];
        }
#pragma unroll
        for (int u = 0; u < HEADS; u++) {
            const int h = g + u * m.groups;
            f2 sq = 0, dot = 0, x[NV][VEC / 2], w[NV][VEC / 2];
#pragma unroll
            for (int k = 0; k < NV; k++) {
                float d[VEC];
                pairs(x_piece[u][k], x[k]);
                d_piece[u][k].values(d);
#pragma unroll
                for (int i = 0; i < VEC / 2; i++) {
                    const float a = d[2 * i], b = d[2 * i + 1];
                    w[k][i] = f2_pack(a * cs[k][i] + b * sn[k][i], b * cs[k][i] - a * sn[k][i]);
                    sq = f2_fma(x[k][i], x[k][i], sq);
                    dot = f2_fma(f2_mul(w[k][i], gain[k][i]), x[k][i], dot);
                }
            }
            const float2 sq2 = f2_get(sq), dot2 = f2_get(dot);
            const float square = group_sum<LOG2>(sq2.x + sq2.y, lanes), product = group_sum<LOG2>(dot2.x + dot2.y, lanes);
            const float r = rsqrtf(square * P.inv_hd + P.eps), f = r * r * (product * P.inv_hd);
            if (!live || h >= m.heads) continue;
#pragma unroll
            for (int k = 0; k < NV; k++) {
                const int c = (lane + k * lanes) * VEC;
                if (c >= hd) break;
                float y[VEC];
#pragma unroll
                for (int i = 0; i < VEC / 2; i++) {
                    const float2 t = f2_get(f2_mul(f2_fma(x[k][i], f2_same(-f), f2_mul(w[k][i], gain[k][i])), f2_same(r)));
                    y[2 * i] = t.x; y[2 * i + 1] = t.y;
                    sum[k][i] = f2_fma(w[k][i], f2_mul(x[k][i], f2_same(r)), sum[k][i]);
                }
                store_either<VEC>(m.out, row * m.ld_out + h * hd + c, m.wide_out, y);
            }
        }
        if (t % FLUSH == FLUSH - 1) flush(false);
    }
    if (!P.partial) return;
    flush(false);
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * hd; c += 256) {
        float s = 0.f;
        for (int o = 0; o < per_block; o++) s += s_gain[o * 2 * hd + c];
        P.partial[(int64_t)blockIdx.x * 2 * hd + c] = s;
    }
}

// dq_gain, dk_gain += the blocks' sums: a block has eight columns (a 32-byte sector), a thread a column and a 64th of the blocks.  SHARED: the two are one tensor
// (queries and keys share their gain), so the thread that adds a column of the queries adds the keys' behind it; apart, the columns of both sides are spread over the
// blocks, which is half a microsecond shorter.
constexpr int FINISH_COLS = 8, FINISH_RUNS = 64;
template <bool SHARED>
__global__ void __launch_bounds__(FINISH_COLS *FINISH_RUNS) gain_finish_kernel(const float *__restrict__ partial, int blocks, int hd, float *dq_gain, float *dk_gain) {
    pdl_wait();
    pdl_next();
    __shared__ float s[FINISH_RUNS][FINISH_COLS];
    const int col = threadIdx.x % FINISH_COLS, run = threadIdx.x / FINISH_COLS, first = blockIdx.x * FINISH_COLS + col;
    for (int side = 0; side < (SHARED ? 2 : 1); side++) {
        const int c = first + side * hd;
        const bool live = first < (SHARED ? hd : 2 * hd);
        float t = 0.f;
        if (live)
#pragma unroll 16
            for (int b = blocks * run / FINISH_RUNS; b < blocks * (run + 1) / FINISH_RUNS; b++) t += partial[(int64_t)b * 2 * hd + c];
        s[run][col] = t;
        __syncthreads();
        if (run == 0 && live) {
            for (int k = 1; k < FINISH_RUNS; k++) t += s[k][col];
            float *to = c < hd ? dq_gain : dk_gain;
            if (to) to[c < hd ? c : c - hd] += t;
        }
        if (SHARED) __syncthreads();
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------------
int launch_status(const char *who) {
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return agpt_set_error(AGPT_E_CUDA, "%s: %s", who, cudaGetErrorString(e));
    return AGPT_OK;
}
int bytes_of(int type) { return type == AGPT_KV_BF16 ? 2 : 4; }
bool type_ok(int t) { return t == AGPT_KV_F32 || t == AGPT_KV_BF16; }

// every row of m starts on a boundary of `vec` elements of its type
bool rows_aligned(const void *p, int64_t ld, int type, int vec) { return !p || (vec::aligned(p, vec * bytes_of(type) > 16 ? 16 : vec * bytes_of(type)) && ld % vec == 0); }

// Heads of a group, whatever their number.  Many heads: four and two, 121 and 193 us at 400k rows of 4 + 4 x 32, 157 and 246 at 40k of 32 + 8 x 128 bfloat16; two and one 129 and
// 228, 197 and 295; one in the forward 144 and 230, four in the backward 208 and 250.  Sides of one or two heads leave places of a group empty: 400k rows of 1 + 1 x 64 135 us, by one
// head a group 76 (backward 143, 121); 200k of 2 + 2 x 64 83, by two 66 (103, by one 119).
constexpr int HEADS = 4, BACK_HEADS = 2, MAX_HEADS = 1024;

void split(Heads &P, int vec, int heads_each, int low) {
    const int pieces = (P.hd + vec - 1) / vec;
    P.lanes_log2 = low < 0 ? 0 : low;
    while (P.lanes_log2 < 5 && (1 << P.lanes_log2) < pieces) P.lanes_log2++;
    P.q.groups = (P.q.heads + heads_each - 1) / heads_each;
    P.k.groups = (P.k.heads + heads_each - 1) / heads_each;
    P.groups = P.q.groups + P.k.groups;
    P.by_groups = vec::Divide((uint32_t)P.groups);
    P.tasks = P.n * P.groups;
}
// Blocks of the backward: as many as run at once, in a number that makes their tasks a multiple of the groups of a row.
int64_t most_blocks(int bytes) { return (int64_t)vec::sm_count() * back_blocks(bytes); }
int backward_blocks(const Heads &P, int bytes) {
    const int per_block = 256 >> P.lanes_log2;
    int step = P.groups;                               // groups / gcd(groups, per_block), per_block a power of two
    for (int b = per_block; b > 1 && step % 2 == 0; b /= 2) step /= 2;
    // two rounds a block at least: a block costs a row of partial sums and its start
    const int64_t want = (P.tasks + 2 * per_block - 1) / (2 * per_block), rounded = (want + step - 1) / step * step, most = most_blocks(bytes) / step * step;
    return (int)(rounded < most ? rounded : most < step ? step : most);
}

// kernel by the lanes of a group (down to 2^LOW; narrower heads leave lanes idle)
template <typename T, int VEC, int NV, int LOW>
int forward(Heads &P, cudaStream_t st) {
    split(P, VEC, HEADS, LOW);
    const int64_t blocks = ((P.tasks << P.lanes_log2) + 255) / 256;
    if (blocks > INT32_MAX) return agpt_set_error(AGPT_E_LIMIT, "qk_norm_rope: too many rows");
    const auto go = [&](void (*kernel)(const Heads)) { pdl_launch(kernel, (unsigned)blocks, 256, 0, st, P); };
    if constexpr (LOW < 0) go(norm_rope_kernel<T, VEC, NV, HEADS, -1>);
    else switch (P.lanes_log2) {
        case 5: go(norm_rope_kernel<T, VEC, NV, HEADS, 5>); break;
        case 4: go(norm_rope_kernel<T, VEC, NV, HEADS, LOW < 4 ? 4 : LOW>); break;
        case 3: go(norm_rope_kernel<T, VEC, NV, HEADS, LOW < 3 ? 3 : LOW>); break;
        case 2: go(norm_rope_kernel<T, VEC, NV, HEADS, LOW < 2 ? 2 : LOW>); break;
        default: go(norm_rope_kernel<T, VEC, NV, HEADS, LOW>);
    }
    return launch_status("qk_norm_rope");
}
template <typename T, typename D, int VEC, int NV, int LOW>
int backward(Heads &P, float *dq_gain, float *dk_gain, cudaStream_t st) {
    split(P, VEC, BACK_HEADS, LOW);
    const int blocks = backward_blocks(P, sizeof(T)), per_block = 256 >> P.lanes_log2;
    const size_t smem = P.partial ? (size_t)per_block * 2 * P.hd * 4 : 0;
    const int64_t row_step = (int64_t)blocks * per_block / P.groups;
    const auto go = [&](void (*kernel)(const Heads, const int64_t)) { pdl_launch(kernel, (unsigned)blocks, 256, smem, st, P, row_step); };
    if constexpr (LOW < 0) go(norm_rope_backward_kernel<T, D, VEC, NV, BACK_HEADS, -1>);
    else switch (P.lanes_log2) {
        case 5: go(norm_rope_backward_kernel<T, D, VEC, NV, BACK_HEADS, 5>); break;
        case 4: go(norm_rope_backward_kernel<T, D, VEC, NV, BACK_HEADS, LOW < 4 ? 4 : LOW>); break;
        case 3: go(norm_rope_backward_kernel<T, D, VEC, NV, BACK_HEADS, LOW < 3 ? 3 : LOW>); break;
        case 2: go(norm_rope_backward_kernel<T, D, VEC, NV, BACK_HEADS, LOW < 2 ? 2 : LOW>); break;
        default: go(norm_rope_backward_kernel<T, D, VEC, NV, BACK_HEADS, LOW>);
    }
    const bool shared = dq_gain == dk_gain;
    if (P.partial) pdl_launch(shared ? gain_finish_kernel<true> : gain_finish_kernel<false>, (unsigned)(((shared ? 1 : 2) * P.hd + FINISH_COLS - 1) / FINISH_COLS),
                              FINISH_COLS * FINISH_RUNS, 0, st, (const float *)P.partial, blocks, P.hd, dq_gain, dk_gain);
    return launch_status("qk_norm_rope_backward");
}

int check(const char *who, int64_t n, int hq, int hk, int hd, int n_pos, int x_type, int64_t q_ld, int64_t k_ld, float eps) {
    if (n < 0 || hq < 1 || hk < 1 || hd < 2 || hd % 2 || n_pos < 1 || !type_ok(x_type) || !(eps > 0.f)) return agpt_set_error(AGPT_E_ARG, "%s: bad argument", who);
    if (hd > 256 || hq + hk > MAX_HEADS) return agpt_set_error(AGPT_E_LIMIT, "%s: head_dim up to 256 and 1024 heads", who);
    if (n > (int64_t)1 << 40) return agpt_set_error(AGPT_E_LIMIT, "%s: too many rows", who);
    if (q_ld < (int64_t)hq * hd || k_ld < (int64_t)hk * hd) return agpt_set_error(AGPT_E_ARG, "%s: rows overlap", who);
    return AGPT_OK;
}

// A head is read whole by the lanes that write it, so an output may lie on what its own side reads, row on row; on anything else it could be written before that is read.
bool same_rows(const vec::Span &a, const vec::Span &b, int64_t n) { return a.p == b.p && a.width == b.width && (a.pitch == b.pitch || n == 1); }
bool may_write(const vec::Span &out, const vec::Span &own, const vec::Span &other, int64_t n) { return (same_rows(out, own, n) || !vec::overlap(out, own, n)) && !vec::overlap(out, other, n); }

}  // namespace

extern "C" int agpt_b200_qk_norm_rope(const void *d_q, int64_t q_ld, const void *d_k, int64_t k_ld, int type, const float *d_q_gain, const float *d_k_gain,
                                      const int32_t *d_pos, const float *d_cos, const float *d_sin, int n_pos, int64_t n, int q_heads, int k_heads, int head_dim,
                                      float eps, void *d_q_out, int64_t q_out_ld, int q_out_type, void *d_k_out, int64_t k_out_ld, int k_out_type, void *stream) {
    if (int rc = check("qk_norm_rope", n, q_heads, k_heads, head_dim, n_pos, type, q_ld, k_ld, eps)) return rc;
    if (!type_ok(q_out_type) || !type_ok(k_out_type) || q_out_ld < (int64_t)q_heads * head_dim || k_out_ld < (int64_t)k_heads * head_dim)
        return agpt_set_error(AGPT_E_ARG, "qk_norm_rope: bad output type or stride");
    if (n == 0) return AGPT_OK;
    if (!d_q || !d_k || !d_pos || !d_cos || !d_sin || !d_q_out || !d_k_out) return agpt_set_error(AGPT_E_ARG, "qk_norm_rope: bad argument");
    const auto span = [&](const void *p, int64_t ld, int heads, int t) { return vec::Span{p, ld * bytes_of(t), (int64_t)heads * head_dim * bytes_of(t)}; };
    const vec::Span q = span(d_q, q_ld, q_heads, type), k = span(d_k, k_ld, k_heads, type), qo = span(d_q_out, q_out_ld, q_heads, q_out_type), ko = span(d_k_out, k_out_ld, k_heads, k_out_type);
    if (!may_write(qo, q, k, n) || !may_write(ko, k, q, n) || vec::overlap(qo, ko, n))
        return agpt_set_error(AGPT_E_ARG, "qk_norm_rope: outputs overlap each other or inputs other than their own");
    Heads P{{d_q, nullptr, d_q_out, q_ld, 0, q_out_ld, d_q_gain, q_out_type == AGPT_KV_F32, q_heads, 0},
            {d_k, nullptr, d_k_out, k_ld, 0, k_out_ld, d_k_gain, k_out_type == AGPT_KV_F32, k_heads, 0},
            d_pos, d_cos, d_sin, n, head_dim, n_pos, 0, 0, eps, 1.f / (float)head_dim, vec::Divide(1), nullptr, 0};
    cudaStream_t st = (cudaStream_t)stream;
    const auto fits = [&](int v) {
        return head_dim % v == 0 && rows_aligned(d_q, q_ld, type, v) && rows_aligned(d_k, k_ld, type, v) && rows_aligned(d_q_out, q_out_ld, q_out_type, v) &&
               rows_aligned(d_k_out, k_out_ld, k_out_type, v) && vec::aligned(d_cos, 16) && vec::aligned(d_sin, 16) && vec::aligned(d_q_gain, 16) && vec::aligned(d_k_gain, 16);
    };
    if (type == AGPT_KV_BF16) return fits(8) ? forward<bf16, 8, 1, 1>(P, st) : forward<bf16, 2, 4, -1>(P, st);
    if (!fits(4)) return forward<float, 2, 4, -1>(P, st);
    return head_dim <= 128 ? forward<float, 4, 1, 2>(P, st) : forward<float, 4, 2, 5>(P, st);
}

extern "C" int64_t agpt_b200_qk_norm_rope_backward_workspace_bytes(int head_dim) {
    if (head_dim < 2 || head_dim > 256) return agpt_set_error(AGPT_E_ARG, "qk_norm_rope_backward_workspace_bytes: bad argument");
    return (most_blocks(4) + MAX_HEADS) * 2 * head_dim * 4;
}

extern "C" int agpt_b200_qk_norm_rope_backward(const void *d_dq, int64_t dq_ld, const void *d_dk, int64_t dk_ld, int grad_type, const void *d_q, int64_t q_ld,
                                               const void *d_k, int64_t k_ld, int type, const float *d_q_gain, const float *d_k_gain, const int32_t *d_pos,
                                               const float *d_cos, const float *d_sin, int n_pos, int64_t n, int q_heads, int k_heads, int head_dim, float eps,
                                               void *d_q_out, int64_t q_out_ld, void *d_k_out, int64_t k_out_ld, float *d_q_gain_grad, float *d_k_gain_grad,
                                               void *d_workspace, int64_t workspace_bytes, void *stream) {
    if (int rc = check("qk_norm_rope_backward", n, q_heads, k_heads, head_dim, n_pos, type, q_ld, k_ld, eps)) return rc;
    const int64_t qc = (int64_t)q_heads * head_dim, kc = (int64_t)k_heads * head_dim;
    if (!type_ok(grad_type) || dq_ld < qc || dk_ld < kc || q_out_ld < qc || k_out_ld < kc) return agpt_set_error(AGPT_E_ARG, "qk_norm_rope_backward: bad type or stride");
    if (n == 0) return AGPT_OK;
    if (!d_dq || !d_dk || !d_q || !d_k || !d_pos || !d_cos || !d_sin || !d_q_out || !d_k_out) return agpt_set_error(AGPT_E_ARG, "qk_norm_rope_backward: bad argument");
    const bool gains = d_q_gain_grad || d_k_gain_grad;
    if (d_q_gain_grad && d_k_gain_grad && d_q_gain_grad != d_k_gain_grad && d_q_gain_grad < d_k_gain_grad + head_dim && d_k_gain_grad < d_q_gain_grad + head_dim)
        return agpt_set_error(AGPT_E_ARG, "qk_norm_rope_backward: gain gradients overlap (one tensor for both, or two apart)");
    if (gains && (!d_workspace || workspace_bytes < agpt_b200_qk_norm_rope_backward_workspace_bytes(head_dim) || !vec::aligned(d_workspace, 16)))
        return agpt_set_error(AGPT_E_ARG, "qk_norm_rope_backward: workspace too small (agpt_b200_qk_norm_rope_backward_workspace_bytes)");
    const auto span = [&](const void *p, int64_t ld, int heads, int t) { return vec::Span{p, ld * bytes_of(t), (int64_t)heads * head_dim * bytes_of(t)}; };
    const vec::Span q = span(d_q, q_ld, q_heads, type), k = span(d_k, k_ld, k_heads, type), qo = span(d_q_out, q_out_ld, q_heads, type), ko = span(d_k_out, k_out_ld, k_heads, type),
                    dq = span(d_dq, dq_ld, q_heads, grad_type), dk = span(d_dk, dk_ld, k_heads, grad_type);
    if (!may_write(qo, q, k, n) || !may_write(qo, dq, dk, n) || !may_write(ko, k, q, n) || !may_write(ko, dk, dq, n) || vec::overlap(qo, ko, n))
        return agpt_set_error(AGPT_E_ARG, "qk_norm_rope_backward: outputs overlap each other or inputs other than their own");
    const int wide = type == AGPT_KV_F32, wide_dy = grad_type == AGPT_KV_F32;
    Heads P{{d_q, d_dq, d_q_out, q_ld, dq_ld, q_out_ld, d_q_gain, wide, q_heads, 0}, {d_k, d_dk, d_k_out, k_ld, dk_ld, k_out_ld, d_k_gain, wide, k_heads, 0},
            d_pos, d_cos, d_sin, n, head_dim, n_pos, 0, 0, eps, 1.f / (float)head_dim, vec::Divide(1), gains ? (float *)d_workspace : nullptr, 0};
    cudaStream_t st = (cudaStream_t)stream;
    const auto fits = [&](int v) {
        return head_dim % v == 0 && rows_aligned(d_q, q_ld, type, v) && rows_aligned(d_k, k_ld, type, v) && rows_aligned(d_q_out, q_out_ld, type, v) &&
               rows_aligned(d_k_out, k_out_ld, type, v) && rows_aligned(d_dq, dq_ld, grad_type, v) && rows_aligned(d_dk, dk_ld, grad_type, v) &&
               vec::aligned(d_cos, 16) && vec::aligned(d_sin, 16) && vec::aligned(d_q_gain, 16) && vec::aligned(d_k_gain, 16);
    };
    const auto run = [&](auto x, auto dy) {
        using T = decltype(x);
        using D = decltype(dy);
        if constexpr (sizeof(T) == 2)
            return fits(8) ? backward<T, D, 8, 1, 1>(P, d_q_gain_grad, d_k_gain_grad, st) : backward<T, D, 2, 4, -1>(P, d_q_gain_grad, d_k_gain_grad, st);
        else if (!fits(4)) return backward<T, D, 2, 4, -1>(P, d_q_gain_grad, d_k_gain_grad, st);
        else return head_dim <= 128 ? backward<T, D, 4, 1, 2>(P, d_q_gain_grad, d_k_gain_grad, st) : backward<T, D, 4, 2, 5>(P, d_q_gain_grad, d_k_gain_grad, st);
    };
    if (wide) return wide_dy ? run(0.f, 0.f) : run(0.f, bf16());
    return wide_dy ? run(bf16(), 0.f) : run(bf16(), bf16());
}
