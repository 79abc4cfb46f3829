// kv_q4.hip -- the paged 4-bit key/value cache: the batch's bookkeeping from its
// lengths (k_kv_plan), rows quantized into the cache (k_kv_store) and read back
// (k_kv_load).  The layout is in qw_kv_q4.hpp.
#include <algorithm>

#include "../../include/qwmoe.h"
#include "qw_kv_q4.hpp"

namespace qw {

namespace {

// ---- plan --------------------------------------------------------------------
//
// Request i holds have = ceil(held / P) pages and needs need = ceil((past + new) / P).
// Prefix sums over the requests of new, of max(0, need - have) and of max(0, have - need)
// say where its token rows start, which entries of the ring of free pages are
// its own and where it puts pages back; every workgroup forms them anew in
// LDS (three ints per request, cheaper than a second launch), then takes its share
// of the token rows, of the new table entries and of the returned pages.  A row's
// page comes from the table where the request already held it, else from the
// ring, so no workgroup waits for another's writes.
struct PlanSeq {
    int n, have, need, grow, give;   // grow: pages wanted; give: pages to put back
    bool good;
};

__device__ __forceinline__ int64_t wave_incl(int64_t v, int lane) {
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t u = __shfl_up(v, o);
        if (lane >= o) v += u;
    }
    return v;
}

__global__ void __launch_bounds__(256) k_kv_plan(KvPlanArgs a) {
    extern __shared__ int32_t s_mem[];
    int32_t* s_start = s_mem;                 // [S + 1] token rows before request i, at most T
    int32_t* s_take = s_start + a.S + 1;      // [S + 1] pages taken before request i
    int32_t* s_give = s_take + a.S + 1;       // [S + 1] pages put back before request i
    __shared__ int64_t s_part[3][4];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int P1 = (1 << a.page_shift) - 1;
    const int64_t head = a.counters[0], tail = a.counters[1];
    const int64_t avail = max((int64_t) 0, min(tail - head, a.n_pages));
    int64_t c_new = 0, c_take = 0, c_give = 0;   // sums over the requests before this round's 256
    int64_t taken = 0;                           // pages of the served requests so far
    bool bad = false, lacking = false;
    for (int base = 0; base < a.S; base += 256) {
        const int i = base + tid;
        int held = 0, past = 0, nn = 0;
        if (i < a.S) {
            held = a.held[i];
            past = a.past[i];
            nn = a.n_new[i];
        }
        const int64_t n = max(nn, 0);
        const int64_t have = ((int64_t) held + P1) >> a.page_shift, need = ((int64_t) past + n + P1) >> a.page_shift;
        const bool sane = held >= 0 && past >= 0 && past <= held && nn >= 0 && have <= a.W && need <= a.W;
        // start, and whether the rows fit
        int64_t v0 = wave_incl(n, lane);
        if (lane == 63) s_part[0][w] = v0;
        __syncthreads();
        for (int u = 0; u < w; ++u) v0 += s_part[0][u];
        const int64_t end = c_new + v0;
        const bool good = i < a.S && sane && end <= a.T;
        int64_t v1 = wave_incl(good ? max(need - have, (int64_t) 0) : 0, lane);
        if (lane == 63) s_part[1][w] = v1;
        __syncthreads();
        for (int u = 0; u < w; ++u) v1 += s_part[1][u];
        const int64_t upto = c_take + v1, grow = good ? max(need - have, (int64_t) 0) : 0;
        const bool served = good && (grow == 0 || upto <= avail);
        int64_t v2 = wave_incl(served ? max(have - need, (int64_t) 0) : 0, lane);
        if (lane == 63) s_part[2][w] = v2;
        __syncthreads();
        for (int u = 0; u < w; ++u) v2 += s_part[2][u];
        const int64_t give = served ? max(have - need, (int64_t) 0) : 0;
        if (i < a.S) {
            s_start[i] = (int32_t) min(end - n, a.T);
            // (a request that is not served: marked by the sign, its prefix is not used)
            s_take[i] = served ? (int32_t) min(upto - grow, a.n_pages) : -1;
            s_give[i] = (int32_t) min(c_give + v2 - give, a.n_pages);
            if (blockIdx.x == 0) {
                a.seq_start[i] = s_start[i];
                a.seq_len[i] = served ? (int32_t) (past + n) : 0;
            }
            bad |= !good;
            lacking |= good && !served;
        }
        c_new += s_part[0][0] + s_part[0][1] + s_part[0][2] + s_part[0][3];
        c_take += s_part[1][0] + s_part[1][1] + s_part[1][2] + s_part[1][3];
        c_give += s_part[2][0] + s_part[2][1] + s_part[2][2] + s_part[2][3];
        // the largest prefix within avail (prefixes ascend, so the served requests' last)
        int64_t t = served && grow > 0 ? upto : 0;
        for (int o = 32; o >= 1; o >>= 1) t = max(t, (int64_t) __shfl_xor(t, o));
        __syncthreads();
        if (lane == 0) s_part[0][w] = t;
        __syncthreads();
        taken = max(max(taken, max(s_part[0][0], s_part[0][1])), max(s_part[0][2], s_part[0][3]));
        __syncthreads();
    }
    const int64_t given = min(c_give, a.n_pages);
    if (tid == 0) {
        s_start[a.S] = (int32_t) min(c_new, a.T);
        s_take[a.S] = (int32_t) taken;
        s_give[a.S] = (int32_t) given;
        if (blockIdx.x == 0) {
            a.seq_start[a.S] = s_start[a.S];
            a.counters_out[0] = head + taken;
            a.counters_out[1] = tail + given;
        }
    }
    if (blockIdx.x == 0 && (bad || lacking))
        atomicOr(a.status, (bad ? QWMOE_STATUS_BAD_SEQ : 0) | (lacking ? QWMOE_STATUS_NO_PAGES : 0));
    __syncthreads();
    auto ring_at = [&](int64_t k) {
        const int64_t r = k % a.n_pages;
        return r < 0 ? r + a.n_pages : r;
    };
    const int64_t g0 = (int64_t) blockIdx.x * 256 + tid, gn = (int64_t) gridDim.x * 256;
    // token rows
    const int n_rows = s_start[a.S];
    for (int64_t r = g0; r < a.T; r += gn) {
        int64_t slot = -1;
        int pos = -1;
        if (r < n_rows) {
            int lo = 0, hi = a.S - 1;   // the first request with s_start[i + 1] > r
            while (lo < hi) {
                const int m = (lo + hi) >> 1;
                if (s_start[m + 1] > r) hi = m;
                else lo = m + 1;
            }
            if (s_take[lo] >= 0) {
                pos = a.past[lo] + (int) (r - s_start[lo]);
                const int p = pos >> a.page_shift, have = (int) (((int64_t) a.held[lo] + P1) >> a.page_shift);
                const int page = p < have ? a.table[lo * a.W + p] : a.ring[ring_at(head + s_take[lo] + (p - have))];
                if (page >= 0 && page < a.n_pages) slot = ((int64_t) page << a.page_shift) + (pos & P1);
                else atomicOr(a.status, QWMOE_STATUS_BAD_SLOT);
            }
        }
        a.slot[r] = slot;
        a.pos[r] = pos;
    }
    // requests' pages: a wave per request
    for (int64_t i = g0 >> 6; i < a.S; i += gn >> 6) {
        if (s_take[i] < 0) continue;
        const int have = (int) (((int64_t) a.held[i] + P1) >> a.page_shift);
        const int need = (int) (((int64_t) a.past[i] + a.n_new[i] + P1) >> a.page_shift);
        for (int p = have + lane; p < need; p += 64)
            a.table[i * a.W + p] = a.ring[ring_at(head + s_take[i] + (p - have))];
        for (int p = need + lane; p < have; p += 64) {
            const int64_t e = s_give[i] + (int64_t) (p - need);
            if (e < a.n_pages) a.ring[ring_at(tail + e)] = a.table[i * a.W + p];
        }
    }
}

// ---- rows ----------------------------------------------------------------------

template <int TYPE>
__device__ __forceinline__ float kv_get(const void* p, int64_t i) {
    if constexpr (TYPE == KV_F32) return ((const float*) p)[i];
    else if constexpr (TYPE == KV_F16) return (float) ((const _Float16*) p)[i];
    else return bitsf((uint32_t) ((const uint16_t*) p)[i] << 16);
}
template <int TYPE>
__device__ __forceinline__ void kv_put(void* p, int64_t i, float v) {
    if constexpr (TYPE == KV_F32) ((float*) p)[i] = v;
    else if constexpr (TYPE == KV_F16) ((_Float16*) p)[i] = (_Float16) v;
    else ((__bf16*) p)[i] = (__bf16) v;
}

// A block's scale: d = f16(m / -8), m the value of largest magnitude (the positive one
// of two), within f16's finite range; a NaN where the block holds one or an infinity.
__device__ __forceinline__ _Float16 kv_scale(float hi, float lo, bool finite) {
    const float m = hi >= -lo ? hi : lo;
    const float d = fminf(fmaxf(m * -0.125f, -65504.0f), 65504.0f);
    return finite ? (_Float16) d : (_Float16) __builtin_nanf("");
}
// x / d to the nearest (ties to even), -8 .. 7, plus 8.  The IEEE quotient of a 24-bit by
// an 11-bit number never rounds onto a border (k + 1/2) d it does not lie on: the border has
// at most 15 significant bits, so x differs from it by a unit of x at least, and the quotient
// by more than half of one of its own.
__device__ __forceinline__ int kv_code(float x, float d) {
    if (d == 0.0f || d != d) return 8;
    return (int) fminf(fmaxf(__builtin_rintf(x / d), -8.0f), 7.0f) + 8;
}

// Eight lanes per block, four values each.
template <int TYPE>
__global__ void __launch_bounds__(256) k_kv_store(KvRowsArgs a) {
    const int NB = a.c.D / 32, per = 2 * a.c.n_head_kv * NB;
    const int64_t id = (int64_t) blockIdx.x * 256 + threadIdx.x, blk = id >> 3;
    const int l = (int) (id & 7);
    const bool in = blk < a.T * per;
    const int64_t t = in ? blk / per : 0;
    const int e = in ? (int) (blk % per) : 0, b = e % NB, hd = e / NB % a.c.n_head_kv;
    const bool value = e / NB >= a.c.n_head_kv;
    float x[4], hi = -INFINITY, lo = INFINITY;
    bool finite = true;
    const char* src = value ? (const char*) a.v + t * a.v_nb1 : (const char*) a.k + t * a.k_nb1;
    for (int j = 0; j < 4; ++j) {
        x[j] = in ? kv_get<TYPE>(src, (int64_t) hd * a.c.D + 32 * b + 4 * l + j) : 0.0f;
        hi = fmaxf(hi, x[j]);
        lo = fminf(lo, x[j]);
        finite &= __builtin_fabsf(x[j]) < INFINITY;
    }
    int fin = finite;
    for (int o = 1; o < 8; o <<= 1) {
        hi = fmaxf(hi, __shfl_xor(hi, o));
        lo = fminf(lo, __shfl_xor(lo, o));
        fin &= __shfl_xor(fin, o);
    }
    const _Float16 d = kv_scale(hi, lo, fin);
    uint32_t key = 0, val = 0;   // this lane's four codes: nibbles of the key dword; one per byte
    for (int j = 0; j < 4; ++j) {
        const uint32_t c = (uint32_t) kv_code(x[j], (float) d);
        const int jj = 4 * (l & 1) + j;
        key |= c << (4 * (jj / 2 + 4 * (jj & 1)));
        val |= c << (8 * j);
    }
    key |= (uint32_t) __shfl_xor((int) key, 1);
    val |= (uint32_t) __shfl_xor((int) val, 4) << 4;   // (lanes 0 .. 3: the dims 16 further on in the high nibbles)
    if (!in) return;
    const int64_t slot = a.slot[t];
    if (slot < 0) return;
    if (slot >> a.c.page_shift >= a.c.n_pages) {
        if (l == 0) atomicOr(a.status, QWMOE_STATUS_BAD_SLOT);
        return;
    }
    uint8_t* cell = a.c.data + a.c.cell(slot) + hd * a.c.head_bytes() + (value ? 18 * a.c.D : 0);
    const int tt = (int) (slot & 15), u = (int) (slot >> 4 & 1), g = tt >> 2, i = tt & 3;
    if (l == 0) ((_Float16*) (cell + 16 * a.c.D))[((4 * u + g) * NB + b) * 4 + i] = d;
    if (!value) {
        if (!(l & 1)) ((uint32_t*) cell)[((16 * u + tt) * 4 + l / 2) * NB + b] = key;
    } else if (l < 4) {
        for (int j = 0; j < 4; ++j)
            cell[((((((b >> 1) * 16 + 4 * l + j) * 4 + g) * 2 + (b & 1)) * 2 + u) * 4) + i] = (uint8_t) (val >> (8 * j));
    }
}

// Eight lanes per block, four values each.
template <int TYPE>
__global__ void __launch_bounds__(256) k_kv_load(KvRowsArgs a) {
    const int NB = a.c.D / 32, per = 2 * a.c.n_head_kv * NB;
    const int64_t id = (int64_t) blockIdx.x * 256 + threadIdx.x, blk = id >> 3;
    const int l = (int) (id & 7);
    if (blk >= a.T * per) return;
    const int64_t t = blk / per;
    const int e = (int) (blk % per), b = e % NB, hd = e / NB % a.c.n_head_kv;
    const bool value = e / NB >= a.c.n_head_kv;
    const int64_t slot = a.slot[t];
    if (slot < 0) return;
    if (slot >> a.c.page_shift >= a.c.n_pages) {
        if (l == 0) atomicOr(a.status, QWMOE_STATUS_BAD_SLOT);
        return;
    }
    const uint8_t* cell = a.c.data + a.c.cell(slot) + hd * a.c.head_bytes() + (value ? 18 * a.c.D : 0);
    const int tt = (int) (slot & 15), u = (int) (slot >> 4 & 1), g = tt >> 2, i = tt & 3;
    const float d = (float) ((const _Float16*) (cell + 16 * a.c.D))[((4 * u + g) * NB + b) * 4 + i];
    char* dst = value ? (char*) a.vo + t * a.v_nb1 : (char*) a.ko + t * a.k_nb1;
    const uint32_t key = value ? 0 : ((const uint32_t*) cell)[((16 * u + tt) * 4 + l / 2) * NB + b];
    for (int j = 0; j < 4; ++j) {
        int c;
        if (!value) {
            const int jj = 4 * (l & 1) + j;
            c = (int) (key >> (4 * (jj / 2 + 4 * (jj & 1)))) & 15;
        } else {
            const int dim = 4 * l + j;
            c = cell[((((((b >> 1) * 16 + (dim & 15)) * 4 + g) * 2 + (b & 1)) * 2 + u) * 4) + i] >> (dim >> 4 << 2) & 15;
        }
        kv_put<TYPE>(dst, (int64_t) hd * a.c.D + 32 * b + 4 * l + j, d * (float) (c - 8));
    }
}

int done() { return hipGetLastError() == hipSuccess ? 0 : -3; }

}  // namespace

int launch_kv_plan(const KvPlanArgs& a, hipStream_t st) {
    if (a.S > KV_MAX_SEQ || a.T >= (int64_t(1) << 31)) return -2;
    const int64_t items = std::max<int64_t>(a.T, (int64_t) a.S * 64);
    const unsigned blocks = (unsigned) std::min<int64_t>((items + 255) / 256, 256);
    hipLaunchKernelGGL(k_kv_plan, dim3(std::max(blocks, 1u)), dim3(256), (size_t) 12 * (a.S + 1), st, a);
    return done();
}

int launch_kv_q4_store(const KvRowsArgs& a, hipStream_t st) {
    const int64_t blocks = (a.T * 2 * a.c.n_head_kv * (a.c.D / 32) * 8 + 255) / 256;
    if (blocks > 0x7fffffff) return -2;
    if (blocks == 0) return 0;
    const dim3 g((unsigned) blocks), b(256);
    if (a.type == KV_F32) hipLaunchKernelGGL(k_kv_store<KV_F32>, g, b, 0, st, a);
    else if (a.type == KV_F16) hipLaunchKernelGGL(k_kv_store<KV_F16>, g, b, 0, st, a);
    else hipLaunchKernelGGL(k_kv_store<KV_BF16>, g, b, 0, st, a);
    return done();
}

int launch_kv_q4_load(const KvRowsArgs& a, hipStream_t st) {
    const int64_t blocks = (a.T * 2 * a.c.n_head_kv * (a.c.D / 32) * 8 + 255) / 256;
    if (blocks > 0x7fffffff) return -2;
    if (blocks == 0) return 0;
    const dim3 g((unsigned) blocks), b(256);
    if (a.type == KV_F32) hipLaunchKernelGGL(k_kv_load<KV_F32>, g, b, 0, st, a);
    else if (a.type == KV_F16) hipLaunchKernelGGL(k_kv_load<KV_F16>, g, b, 0, st, a);
    else hipLaunchKernelGGL(k_kv_load<KV_BF16>, g, b, 0, st, a);
    return done();
}

}  // namespace qw
