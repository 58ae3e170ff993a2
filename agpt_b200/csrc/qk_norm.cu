// RMS norm of queries and keys per head and their rotation by position, in one pass over the rows, forward and backward.
//
//   r = 1 / sqrt(mean(x^2) + eps)   u = r x   y = R(pos) (g u)        for every row and head, g the gain of queries or of keys
//   w = R(pos)^T dy   c = g w       dx = r (c - u mean(c u))          dg += sum over rows and heads of w u
//
// The pairs (2 i, 2 i + 1) of a head turn by the entries 2 i of the tables, as in agpt_b200_rope.  The backward forms r again from x, so the
// forward keeps nothing.  Statistics and sums are float32; bfloat16 rows are rounded once, on the way out.
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/agpt_b200.h"
#include "internal.h"
#include "pdl.cuh"
#include "vec.cuh"

namespace {

using bf16 = __nv_bfloat16;

struct Rows {                          // queries or keys: heads * head_dim columns, rows ld elements apart
    const void *x, *dy;
    void *out;                         // y, or dx
    int64_t ld_x, ld_dy, ld_out;
    const float *gain;                 // NULL: 1
    int wide_out, wide_dy;             // out, dy are float32 (else bfloat16)
};
struct Heads {
    Rows q, k;
    const int32_t *pos;
    const float *cosv, *sinv;
    int64_t n;
    int hq, hk, hd, n_pos, lanes_log2, groups;      // groups of lanes per row, HEADS heads each
    float eps;
    vec::Divide by_groups;
    float *partial;                    // backward: [blocks][2][hd]
    int64_t tasks;
};

__device__ __forceinline__ float group_sum(float v, int lanes) {
    for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
template <int VEC> __device__ __forceinline__ void load_either(const void *p, int64_t at, int wide, float (&v)[VEC]) {
    if (wide) vec::load<VEC>(reinterpret_cast<const float *>(p) + at, v);
    else vec::load<VEC>(reinterpret_cast<const bf16 *>(p) + at, v);
}
template <int VEC> __device__ __forceinline__ void store_either(void *p, int64_t at, int wide, const float (&v)[VEC]) {
    if (wide) vec::store<VEC>(reinterpret_cast<float *>(p) + at, v);
    else vec::store<VEC>(reinterpret_cast<bf16 *>(p) + at, v);
}
// pair i of VEC elements: cos and sin
template <int VEC> __device__ __forceinline__ void load_table(const float *p, float (&v)[VEC / 2]) {
    if constexpr (VEC % 4 == 0) {
#pragma unroll
        for (int i = 0; i < VEC / 4; i++) {
            const float4 x = __ldg(reinterpret_cast<const float4 *>(p) + i);
            v[2 * i] = x.x; v[2 * i + 1] = x.z;
        }
    } else {
#pragma unroll
        for (int i = 0; i < VEC / 2; i++) v[i] = __ldg(p + 2 * i);
    }
}

// A group of lanes owns HEADS heads of a row, `groups` apart, so that neighbouring groups read neighbouring heads and the table's entries
// are read once for HEADS heads; a lane has NV pieces of VEC columns, `lanes` pieces apart.
template <typename T, int VEC, int NV, int HEADS>
__global__ void __launch_bounds__(256) norm_rope_kernel(const __grid_constant__ Heads P) {
    pdl_wait();
    pdl_next();
    const int lanes = 1 << P.lanes_log2, lane = threadIdx.x & (lanes - 1);
    const int64_t task = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> P.lanes_log2;
    const bool live = task < P.tasks;
    const int64_t row = live ? vec::quotient(task, P.by_groups) : 0;
    const int g = (int)(live ? task - row * P.groups : 0), hd = P.hd, heads = P.hq + P.hk;
    float v[HEADS][NV][VEC];
#pragma unroll
    for (int u = 0; u < HEADS; u++) {
        const int h = g + u * P.groups;
        const bool is_q = h < P.hq;
        const Rows &m = is_q ? P.q : P.k;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int c = (lane + k * lanes) * VEC;
            if (live && h < heads && c < hd) vec::load<VEC>(reinterpret_cast<const T *>(m.x) + row * m.ld_x + (is_q ? h : h - P.hq) * hd + c, v[u][k]);
            else
#pragma unroll
                for (int i = 0; i < VEC; i++) v[u][k][i] = 0.f;
        }
    }
    float cs[NV][VEC / 2], sn[NV][VEC / 2];
    const int at = live ? min(max(__ldg(P.pos + row), 0), P.n_pos - 1) : 0;
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int c = (lane + k * lanes) * VEC;
        if (c < hd) {
            load_table<VEC>(P.cosv + (int64_t)at * hd + c, cs[k]);
            load_table<VEC>(P.sinv + (int64_t)at * hd + c, sn[k]);
        }
    }
    float r[HEADS];
#pragma unroll
    for (int u = 0; u < HEADS; u++) {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int i = 0; i < VEC; i++) s += v[u][k][i] * v[u][k][i];
        r[u] = 1.f / sqrtf(group_sum(s, lanes) / (float)hd + P.eps);
    }
    if (!live) return;
#pragma unroll
    for (int u = 0; u < HEADS; u++) {
        const int h = g + u * P.groups;
        if (h >= heads) break;
        const bool is_q = h < P.hq;
        const Rows &m = is_q ? P.q : P.k;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int c = (lane + k * lanes) * VEC;
            if (c >= hd) break;
            float y[VEC];
#pragma unroll
            for (int i = 0; i < VEC; i += 2) {
                const float a = v[u][k][i] * r[u] * (m.gain ? __ldg(m.gain + c + i) : 1.f), b = v[u][k][i + 1] * r[u] * (m.gain ? __ldg(m.gain + c + i + 1) : 1.f);
                y[i] = a * cs[k][i / 2] - b * sn[k][i / 2];
                y[i + 1] = a * sn[k][i / 2] + b * cs[k][i / 2];
            }
            store_either<VEC>(m.out, row * m.ld_out + (is_q ? h : h - P.hq) * hd + c, m.wide_out, y);
        }
    }
}

// A thread keeps its columns' gain gradients over all rows of its group; the block adds its groups in order into partial[block].
template <typename T, int VEC, int NV, int HEADS>
__global__ void __launch_bounds__(256) norm_rope_backward_kernel(const __grid_constant__ Heads P) {
    pdl_wait();
    pdl_next();
    extern __shared__ float s_gain[];                  // [groups of the block][2][hd]
    const int lanes = 1 << P.lanes_log2, lane = threadIdx.x & (lanes - 1), per_block = 256 >> P.lanes_log2, own = threadIdx.x >> P.lanes_log2;
    const int hd = P.hd, heads = P.hq + P.hk;
    float sum[2][NV][VEC];
#pragma unroll
    for (int w = 0; w < 2; w++)
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int i = 0; i < VEC; i++) sum[w][k][i] = 0.f;
    const int64_t rounds = (P.tasks + (int64_t)gridDim.x * per_block - 1) / ((int64_t)gridDim.x * per_block);
    for (int64_t t = 0; t < rounds; t++) {
        const int64_t task = (t * gridDim.x + blockIdx.x) * per_block + own;
        const bool live = task < P.tasks;
        const int64_t row = live ? vec::quotient(task, P.by_groups) : 0;
        const int g = (int)(live ? task - row * P.groups : 0);
        float x[HEADS][NV][VEC], d[HEADS][NV][VEC];
#pragma unroll
        for (int u = 0; u < HEADS; u++) {
            const int h = g + u * P.groups;
            const bool is_q = h < P.hq;
            const Rows &m = is_q ? P.q : P.k;
#pragma unroll
            for (int k = 0; k < NV; k++) {
                const int c = (lane + k * lanes) * VEC;
                if (live && h < heads && c < hd) {
                    const int col = (is_q ? h : h - P.hq) * hd + c;
                    vec::load<VEC>(reinterpret_cast<const T *>(m.x) + row * m.ld_x + col, x[u][k]);
                    load_either<VEC>(m.dy, row * m.ld_dy + col, m.wide_dy, d[u][k]);
                } else
#pragma unroll
                    for (int i = 0; i < VEC; i++) x[u][k][i] = d[u][k][i] = 0.f;
            }
        }
        const int at = live ? min(max(__ldg(P.pos + row), 0), P.n_pos - 1) : 0;
        float cs[NV][VEC / 2], sn[NV][VEC / 2];
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int c = (lane + k * lanes) * VEC;
            if (c < hd) {
                load_table<VEC>(P.cosv + (int64_t)at * hd + c, cs[k]);
                load_table<VEC>(P.sinv + (int64_t)at * hd + c, sn[k]);
            }
        }
#pragma unroll
        for (int u = 0; u < HEADS; u++) {
            const int h = g + u * P.groups;
            const bool is_q = h < P.hq;
            const Rows &m = is_q ? P.q : P.k;
            float sq = 0.f, dot = 0.f, w[NV][VEC];
#pragma unroll
            for (int k = 0; k < NV; k++) {
                const int c = (lane + k * lanes) * VEC;
#pragma unroll
                for (int i = 0; i < VEC; i += 2) {
                    const float a = d[u][k][i], b = d[u][k][i + 1], co = c < hd ? cs[k][i / 2] : 0.f, si = c < hd ? sn[k][i / 2] : 0.f;
                    w[k][i] = a * co + b * si;
                    w[k][i + 1] = b * co - a * si;
                }
#pragma unroll
                for (int i = 0; i < VEC; i++) {
                    sq += x[u][k][i] * x[u][k][i];
                    d[u][k][i] = w[k][i] * (m.gain && c < hd ? __ldg(m.gain + c + i) : 1.f);
                    dot += d[u][k][i] * x[u][k][i];
                }
            }
            sq = group_sum(sq, lanes);
            dot = group_sum(dot, lanes);
            const float r = 1.f / sqrtf(sq / (float)hd + P.eps), f = r * r * (dot / (float)hd);
            if (!live || h >= heads) continue;
#pragma unroll
            for (int k = 0; k < NV; k++) {
                const int c = (lane + k * lanes) * VEC;
                if (c >= hd) break;
                float y[VEC];
#pragma unroll
                for (int i = 0; i < VEC; i++) {
                    y[i] = r * (d[u][k][i] - x[u][k][i] * f);
                    const float e = w[k][i] * (x[u][k][i] * r);
                    if (is_q) sum[0][k][i] += e; else sum[1][k][i] += e;
                }
                store_either<VEC>(m.out, row * m.ld_out + (is_q ? h : h - P.hq) * hd + c, m.wide_out, y);
            }
        }
    }
    if (!P.partial) return;
#pragma unroll
    for (int w = 0; w < 2; w++)
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int c = (lane + k * lanes) * VEC;
            if (c < hd)
#pragma unroll
                for (int i = 0; i < VEC; i++) s_gain[(own * 2 + w) * hd + c + i] = sum[w][k][i];
        }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * hd; c += 256) {
        float s = 0.f;
        for (int o = 0; o < per_block; o++) s += s_gain[o * 2 * hd + c];
        P.partial[(int64_t)blockIdx.x * 2 * hd + c] = s;
    }
}

// dq_gain, dk_gain += the blocks' sums: a block has 32 columns, its eight warps a run of the blocks each
__global__ void __launch_bounds__(256) gain_finish_kernel(const float *__restrict__ partial, int blocks, int hd, float *__restrict__ dq_gain, float *__restrict__ dk_gain) {
    pdl_wait();
    pdl_next();
    __shared__ float s[8][32];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float t = 0.f;
    if (c < 2 * hd)
#pragma unroll 8
        for (int b = blocks * w / 8; b < blocks * (w + 1) / 8; b++) t += partial[(int64_t)b * 2 * hd + c];
    s[w][lane] = t;
    __syncthreads();
    if (w || c >= 2 * hd) return;
    for (int k = 1; k < 8; k++) t += s[k][lane];
    float *to = c < hd ? dq_gain : dk_gain;
    if (to) to[c < hd ? c : c - hd] += t;
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

constexpr int HEADS = 4, BACK_HEADS = 2;

void split(Heads &P, int vec, int heads_each) {
    const int pieces = (P.hd + vec - 1) / vec;
    P.lanes_log2 = 0;
    while (P.lanes_log2 < 5 && (1 << P.lanes_log2) < pieces) P.lanes_log2++;
    P.groups = (P.hq + P.hk + heads_each - 1) / heads_each;
    P.by_groups = vec::Divide((uint32_t)P.groups);
    P.tasks = P.n * P.groups;
}
int backward_blocks(int64_t tasks, int lanes_log2) {
    const int64_t want = (tasks + (256 >> lanes_log2) - 1) / (256 >> lanes_log2), most = (int64_t)vec::sm_count() * 4;
    return (int)(want < most ? want : most);
}

template <typename T, int VEC, int NV>
int forward(Heads &P, cudaStream_t st) {
    split(P, VEC, HEADS);
    const int64_t blocks = ((P.tasks << P.lanes_log2) + 255) / 256;
    if (blocks > INT32_MAX) return agpt_set_error(AGPT_E_LIMIT, "qk_norm_rope: too many rows");
    pdl_launch(norm_rope_kernel<T, VEC, NV, HEADS>, (unsigned)blocks, 256, 0, st, P);
    return launch_status("qk_norm_rope");
}
template <typename T, int VEC, int NV>
int backward(Heads &P, float *dq_gain, float *dk_gain, cudaStream_t st) {
    split(P, VEC, BACK_HEADS);
    const int blocks = backward_blocks(P.tasks, P.lanes_log2);
    const size_t smem = P.partial ? (size_t)(256 >> P.lanes_log2) * 2 * P.hd * 4 : 0;
    pdl_launch(norm_rope_backward_kernel<T, VEC, NV, BACK_HEADS>, (unsigned)blocks, 256, smem, st, P);
    if (P.partial) pdl_launch(gain_finish_kernel, (unsigned)((2 * P.hd + 31) / 32), 256, 0, st, (const float *)P.partial, blocks, P.hd, dq_gain, dk_gain);
    return launch_status("qk_norm_rope_backward");
}

int check(const char *who, int64_t n, int hq, int hk, int hd, int n_pos, int x_type, int64_t q_ld, int64_t k_ld, float eps) {
    if (n < 0 || hq < 1 || hk < 1 || hd < 2 || hd % 2 || n_pos < 1 || !type_ok(x_type) || !(eps > 0.f)) return agpt_set_error(AGPT_E_ARG, "%s: bad argument", who);
    if (hd > 256 || hq + hk > 1024) return agpt_set_error(AGPT_E_LIMIT, "%s: head_dim up to 256 and 1024 heads", who);
    if (n > (int64_t)1 << 40) return agpt_set_error(AGPT_E_LIMIT, "%s: too many rows", who);
    if (q_ld < (int64_t)hq * hd || k_ld < (int64_t)hk * hd) return agpt_set_error(AGPT_E_ARG, "%s: rows overlap", who);
    return AGPT_OK;
}

}  // namespace

extern "C" int agpt_b200_qk_norm_rope(const void *d_q, int64_t q_ld, const void *d_k, int64_t k_ld, int type, const float *d_q_gain, const float *d_k_gain,
                                      const int32_t *d_pos, const float *d_cos, const float *d_sin, int n_pos, int64_t n, int q_heads, int k_heads, int head_dim,
                                      float eps, void *d_q_out, int64_t q_out_ld, int q_out_type, void *d_k_out, int64_t k_out_ld, int k_out_type, void *stream) {
    if (int rc = check("qk_norm_rope", n, q_heads, k_heads, head_dim, n_pos, type, q_ld, k_ld, eps)) return rc;
    if (!type_ok(q_out_type) || !type_ok(k_out_type) || q_out_ld < (int64_t)q_heads * head_dim || k_out_ld < (int64_t)k_heads * head_dim)
        return agpt_set_error(AGPT_E_ARG, "qk_norm_rope: bad output type or stride");
    if (n == 0) return AGPT_OK;
    if (!d_q || !d_k || !d_pos || !d_cos || !d_sin || !d_q_out || !d_k_out) return agpt_set_error(AGPT_E_ARG, "qk_norm_rope: bad argument");
    Heads P{{d_q, nullptr, d_q_out, q_ld, 0, q_out_ld, d_q_gain, q_out_type == AGPT_KV_F32, 0},
            {d_k, nullptr, d_k_out, k_ld, 0, k_out_ld, d_k_gain, k_out_type == AGPT_KV_F32, 0},
            d_pos, d_cos, d_sin, n, q_heads, k_heads, head_dim, n_pos, 0, 0, eps, vec::Divide(1), nullptr, 0};
    cudaStream_t st = (cudaStream_t)stream;
    const auto fits = [&](int v) {
        return head_dim % v == 0 && rows_aligned(d_q, q_ld, type, v) && rows_aligned(d_k, k_ld, type, v) && rows_aligned(d_q_out, q_out_ld, q_out_type, v) &&
               rows_aligned(d_k_out, k_out_ld, k_out_type, v) && vec::aligned(d_cos, 16) && vec::aligned(d_sin, 16);
    };
    if (type == AGPT_KV_BF16) return fits(8) ? forward<bf16, 8, 1>(P, st) : forward<bf16, 2, 4>(P, st);
    if (!fits(4)) return forward<float, 2, 4>(P, st);
    return head_dim <= 128 ? forward<float, 4, 1>(P, st) : forward<float, 4, 2>(P, st);
}

extern "C" int64_t agpt_b200_qk_norm_rope_backward_workspace_bytes(int head_dim) {
    if (head_dim < 2 || head_dim > 256) return agpt_set_error(AGPT_E_ARG, "qk_norm_rope_backward_workspace_bytes: bad argument");
    return (int64_t)vec::sm_count() * 4 * 2 * head_dim * 4;
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
    if (gains && (!d_workspace || workspace_bytes < agpt_b200_qk_norm_rope_backward_workspace_bytes(head_dim) || !vec::aligned(d_workspace, 16)))
        return agpt_set_error(AGPT_E_ARG, "qk_norm_rope_backward: workspace too small (agpt_b200_qk_norm_rope_backward_workspace_bytes)");
    const int wide = type == AGPT_KV_F32, wide_dy = grad_type == AGPT_KV_F32;
    Heads P{{d_q, d_dq, d_q_out, q_ld, dq_ld, q_out_ld, d_q_gain, wide, wide_dy}, {d_k, d_dk, d_k_out, k_ld, dk_ld, k_out_ld, d_k_gain, wide, wide_dy},
            d_pos, d_cos, d_sin, n, q_heads, k_heads, head_dim, n_pos, 0, 0, eps, vec::Divide(1), gains ? (float *)d_workspace : nullptr, 0};
    cudaStream_t st = (cudaStream_t)stream;
    const auto fits = [&](int v) {
        return head_dim % v == 0 && rows_aligned(d_q, q_ld, type, v) && rows_aligned(d_k, k_ld, type, v) && rows_aligned(d_q_out, q_out_ld, type, v) &&
               rows_aligned(d_k_out, k_out_ld, type, v) && rows_aligned(d_dq, dq_ld, grad_type, v) && rows_aligned(d_dk, dk_ld, grad_type, v) &&
               vec::aligned(d_cos, 16) && vec::aligned(d_sin, 16);
    };
    if (type == AGPT_KV_BF16)
        return fits(8) ? backward<bf16, 8, 1>(P, d_q_gain_grad, d_k_gain_grad, st) : backward<bf16, 2, 4>(P, d_q_gain_grad, d_k_gain_grad, st);
    if (!fits(4)) return backward<float, 2, 4>(P, d_q_gain_grad, d_k_gain_grad, st);
    return head_dim <= 128 ? backward<float, 4, 1>(P, d_q_gain_grad, d_k_gain_grad, st) : backward<float, 4, 2>(P, d_q_gain_grad, d_k_gain_grad, st);
}
