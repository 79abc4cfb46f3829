// attn_q4.hip -- causal attention of a batch of requests over the paged 4-bit cache
// (layout in qw_kv_q4.hpp): row (token t of n, query head h) of request i sees its keys
// 0 .. len - n + t,
//   o = sum_j softmax_j(scale q . k_j) v_j.
#include "../../include/qwmoe.h"
#include "qw_kv_q4.hpp"

namespace qw {

namespace {

template <int TYPE>
__device__ __forceinline__ float q4_get(const void* p, int64_t i) {
    if constexpr (TYPE == KV_F32) return ((const float*) p)[i];
    else if constexpr (TYPE == KV_F16) return (float) ((const _Float16*) p)[i];
    else return bitsf((uint32_t) ((const uint16_t*) p)[i] << 16);
}
template <int TYPE>
__device__ __forceinline__ void q4_put(void* p, int64_t i, float v) {
    if constexpr (TYPE == KV_F32) ((float*) p)[i] = v;
    else if constexpr (TYPE == KV_F16) ((_Float16*) p)[i] = (_Float16) v;
    else ((__bf16*) p)[i] = (__bf16) v;
}

__device__ __forceinline__ float block_max(float v, float* s) {
    for (int o = 32; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    return fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
}
__device__ __forceinline__ float block_sum(float v, float* s) {
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    return (s[0] + s[1]) + (s[2] + s[3]);
}

// A workgroup per (token row, head): 256 keys at a time, a thread forms a key's score,
// then a thread per dimension adds the values, the running maximum and sum rescaled.
template <int TYPE>
__global__ void __launch_bounds__(256) k_attn_q4(AttnQ4Args a) {
    __shared__ float s_q[256], s_p[256], s_r[4];
    const int tid = threadIdx.x, D = a.c.D, NB = D / 32, h = blockIdx.y, g = h / (a.n_head / a.c.n_head_kv);
    const int64_t r = blockIdx.x;
    int i = 0;
    while (i < a.S && a.seq_start[i + 1] <= r) ++i;
    if (i == a.S || a.seq_start[i] > r) return;
    const int n = a.seq_start[i + 1] - a.seq_start[i];
    int len = a.seq_len[i];
    if (len < 0 || len > a.max_len || n > a.max_new || len > a.W << a.c.page_shift) {
        len = 0;
        if (tid == 0) atomicOr(a.status, QWMOE_STATUS_BAD_SEQ);
    }
    const int seen = min(len, len - n + (int) (r - a.seq_start[i]) + 1);
    if (tid < D) s_q[tid] = q4_get<TYPE>((const char*) a.q + r * a.q_nb1, (int64_t) h * D + tid) * a.scale;
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    for (int k0 = 0; k0 < seen; k0 += 256) {
        const int k = k0 + tid;
        auto cell_of = [&](int key) -> const uint8_t* {
            const int page = a.table[i * a.W + (key >> a.c.page_shift)];
            if (page < 0 || page >= a.c.n_pages) return nullptr;
            return a.c.data + a.c.cell(((int64_t) page << a.c.page_shift) + (key & ((1 << a.c.page_shift) - 1))) +
                   g * a.c.head_bytes();
        };
        __syncthreads();
        float sc = -INFINITY;
        if (k < seen) {
            const uint8_t* cell = cell_of(k);
            if (!cell) atomicOr(a.status, QWMOE_STATUS_BAD_SLOT);
            else {
                const int tt = k & 15, u = k >> 4 & 1;
                sc = 0.0f;
                for (int b = 0; b < NB; ++b) {
                    float s = 0.0f;
                    for (int q = 0; q < 4; ++q) {
                        const uint32_t w = ((const uint32_t*) cell)[((16 * u + tt) * 4 + q) * NB + b];
                        for (int j = 0; j < 8; ++j)
                            s += s_q[32 * b + 8 * q + j] * (float) ((int) (w >> (4 * (j / 2 + 4 * (j & 1))) & 15) - 8);
                    }
                    sc += s * (float) ((const _Float16*) (cell + 16 * D))[((4 * u + (tt >> 2)) * NB + b) * 4 + (tt & 3)];
                }
            }
        }
        const float mn = fmaxf(m, block_max(sc, s_r)), mu = mn == -INFINITY ? 0.0f : mn;
        const float f = exp2f(m - mu), p = exp2f(sc - mu);
        s_p[tid] = p;
        l = l * f + block_sum(p, s_r);
        o *= f;
        m = mn;
        if (tid < D) {
            const int b = tid >> 5, e = tid & 31;
            for (int j = 0; j < 256 && k0 + j < seen; ++j) {
                const uint8_t* cell = cell_of(k0 + j);
                if (!cell) continue;
                cell += 18 * D;
                const int tt = j & 15, u = j >> 4 & 1;
                const int c = cell[((((((b >> 1) * 16 + (e & 15)) * 4 + (tt >> 2)) * 2 + (b & 1)) * 2 + u) * 4) + (tt & 3)] >>
                                  (e >> 4 << 2) & 15;
                const float d = (float) ((const _Float16*) (cell + 16 * D))[((4 * u + (tt >> 2)) * NB + b) * 4 + (tt & 3)];
                o += s_p[j] * (d * (float) (c - 8));
            }
        }
    }
    if (tid < D) q4_put<TYPE>((char*) a.out + r * a.out_nb1, (int64_t) h * D + tid, l == 0.0f ? 0.0f : o / l);
}

}  // namespace

int launch_attn_q4(const AttnQ4Args& a, hipStream_t st) {
    if (a.T == 0 || a.S == 0) return 0;
    const dim3 g((unsigned) a.T, (unsigned) a.n_head);
    if (a.type == KV_F32) hipLaunchKernelGGL(k_attn_q4<KV_F32>, g, dim3(256), 0, st, a);
    else if (a.type == KV_F16) hipLaunchKernelGGL(k_attn_q4<KV_F16>, g, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(k_attn_q4<KV_BF16>, g, dim3(256), 0, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -3;
}

}  // namespace qw
