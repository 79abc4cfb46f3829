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
// A few kilobytes: what it takes is the chain counters -> three scans -> row's search -> page -> slot,
// so the scans stay in registers (DPP adds, one LDS exchange each).  One decode step of 24
// requests 3.9 us, a round of 512 with 3000 tokens' prompts 6.3 (with 64-bit shuffles
// 5.0 and 8.6); an empty kernel takes 1.4.
__global__ void __launch_bounds__(256) k_kv_plan(KvPlanArgs a) {
    extern __shared__ int32_t s_mem[];
    int32_t* s_start = s_mem;                 // [S + 1] token rows before request i, at most T
    int32_t* s_take = s_start + a.S + 1;      // [S + 1] pages taken before request i
    int32_t* s_give = s_take + a.S + 1;       // [S + 1] pages put back before request i
    __shared__ uint32_t s_part[4][4];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int P1 = (1 << a.page_shift) - 1;
    const int64_t head = a.counters[0], tail = a.counters[1];
    const uint32_t avail = (uint32_t) max((int64_t) 0, min(tail - head, a.n_pages));
    uint32_t c_new = 0, c_take = 0, c_give = 0;   // sums over the requests before this round's 256
    uint32_t taken = 0;                           // pages of the served requests so far
    bool bad = false, lacking = false;
    // the sum up to this lane over the round, on top of c; c takes the round's
    auto scan = [&](uint32_t v, uint32_t& c, uint32_t* part) {
        v = kv_wave_incl(v);
        if (lane == 63) part[w] = v;
        __syncthreads();
        uint32_t before = c;
        for (int u = 0; u < 4; ++u) {
            if (u < w) before = kv_add(before, part[u]);
            c = kv_add(c, part[u]);
        }
        return kv_add(before, v);
    };
    for (int base = 0; base < a.S; base += 256) {
        const int i = base + tid;
        int held = 0, past = 0, nn = 0;
        if (i < a.S) {
            held = a.held[i];
            past = a.past[i];
            nn = a.n_new[i];
        }
        const uint32_t n = (uint32_t) max(nn, 0);
        const int64_t have = ((int64_t) held + P1) >> a.page_shift, need = ((int64_t) past + n + P1) >> a.page_shift;
        const bool sane = held >= 0 && past >= 0 && past <= held && nn >= 0 && have <= a.W && need <= a.W;
        // start, and whether the rows fit
        const uint32_t end = scan(n, c_new, s_part[0]);
        const bool good = i < a.S && sane && end <= (uint32_t) a.T;
        const uint32_t grow = good ? (uint32_t) max(need - have, (int64_t) 0) : 0;
        const uint32_t upto = scan(grow, c_take, s_part[1]);
        const bool served = good && (grow == 0 || upto <= avail);
        const uint32_t give = served ? (uint32_t) max(have - need, (int64_t) 0) : 0;
        const uint32_t back = scan(give, c_give, s_part[2]);
        if (i < a.S) {
            s_start[i] = (int32_t) min(end - n, (uint32_t) a.T);
            // (a request that is not served: marked by the sign, its prefix is not used)
            s_take[i] = served ? (int32_t) min(upto - grow, (uint32_t) a.n_pages) : -1;
            s_give[i] = (int32_t) min(back - give, (uint32_t) a.n_pages);
            if (blockIdx.x == 0) {
                a.seq_start[i] = s_start[i];
                a.seq_len[i] = served ? (int32_t) (past + n) : 0;
            }
            bad |= !good;
            lacking |= good && !served;
        }
        // the largest prefix within avail (prefixes ascend, so the served requests' last)
        uint32_t t = served && grow > 0 ? upto : 0;
        t = max(t, kv_dpp<0x111>(t));
        t = max(t, kv_dpp<0x112>(t));
        t = max(t, kv_dpp<0x114>(t));
        t = max(t, kv_dpp<0x118>(t));
        t = max(t, kv_dpp<0x142, 0xA>(t));
        t = max(t, kv_dpp<0x143, 0xC>(t));
        if (lane == 63) s_part[3][w] = t;
        __syncthreads();
        for (int u = 0; u < 4; ++u) taken = max(taken, s_part[3][u]);
        // (the next round writes s_part[0] while slower waves still read s_part[3]: others' words)
    }
    const uint32_t given = min(c_give, (uint32_t) a.n_pages);
    if (tid == 0) {
        s_start[a.S] = (int32_t) min(c_new, (uint32_t) a.T);
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
//
// Both move each row and each cell once: bytes bound them, and below a few thousand rows the
// chain slot -> cell -> row.  A workgroup has 16 rows of one head, keys (blockIdx.y even) or
// values, and PB of their blocks.  On the rows' side eight lanes share a block of 32 dims,
// four each, so that a wave touches up to 1 KiB of whole rows; on the cell's side a key's dwords
// are dense per token, but a value's bytes lie among those of 32 tokens.  They go through LDS,
// and there the token runs with the lane: rows of consecutive places put the bytes of a
// line into one instruction.  Measured against lanes that read and wrote their bytes
// where they lie: 20000 rows of four heads of 128 out to f32 17.1 us (93 MB, 5.5 TB/s), was 36.8;
// 4133 bf16 rows in 7.1 us, was 13.6, out 6.8, was 9.2; 24 f32 rows in 2.9 and out 3.2.
// 32 rows a workgroup: 3.5 and 3.7 for the 24, 19.2 for the 20000 (16: 20.4, both with ordinary stores).
constexpr int KV_ROWS = 16;

// four dims 4 n .. 4 n + 3 of a row, aligned as their type
template <int TYPE>
__device__ __forceinline__ void kv_get4(const char* row, int n, float (&x)[4]) {
    if constexpr (TYPE == KV_F32) {
        __builtin_memcpy(x, row + 16 * n, 16);
    } else {
        uint16_t h[4];
        __builtin_memcpy(h, row + 8 * n, 8);
        for (int j = 0; j < 4; ++j) {
            if constexpr (TYPE == KV_F16) x[j] = (float) __builtin_bit_cast(_Float16, h[j]);
            else x[j] = bitsf((uint32_t) h[j] << 16);
        }
    }
}
// (Rows read back go out past the caches: a large output leaves them to the cells.  20000 rows of
// four heads of 128 in f32: 17.1 us so, 20.4 with ordinary stores; 77 rows: 3.3 both.)
template <int TYPE>
__device__ __forceinline__ void kv_put4(char* row, int n, const float (&x)[4]) {
    if constexpr (TYPE == KV_F32) {
        typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
        __builtin_nontemporal_store(vec{x[0], x[1], x[2], x[3]}, (vec*) (row + 16 * n));
    } else {
        typedef uint16_t vec __attribute__((ext_vector_type(4), aligned(2)));
        uint16_t h[4];
        for (int j = 0; j < 4; ++j) {
            if constexpr (TYPE == KV_F16) h[j] = __builtin_bit_cast(uint16_t, (_Float16) x[j]);
            else h[j] = __builtin_bit_cast(uint16_t, (__bf16) x[j]);
        }
        __builtin_nontemporal_store(vec{h[0], h[1], h[2], h[3]}, (vec*) (row + 8 * n));
    }
}

// Ordered by magnitude, the positive one of two above the negative; 0xff000000 and up: not finite.
__device__ __forceinline__ uint32_t kv_rank(float x) {
    const uint32_t v = fbits(x);
    return (v << 1 | v >> 31) ^ 1;
}
// the largest of eight lanes
__device__ __forceinline__ uint32_t kv_top8(uint32_t v) {
    v = max(v, kv_dpp<0xB1>(v));          // neighbours
    v = max(v, kv_dpp<0x4E>(v));          // pairs
    return max(v, kv_dpp<0x141>(v));      // the quads of eight lanes (mirrored)
}
// A block's scale: d = f16(m / -8), m the value of largest magnitude, within f16's finite
// range; a NaN where the block holds one or an infinity.
__device__ __forceinline__ _Float16 kv_scale(uint32_t rank) {
    const float m = bitsf((rank >> 1 | rank << 31) ^ 0x80000000u);
    const float d = fminf(fmaxf(m * -0.125f, -65504.0f), 65504.0f);
    return rank < 0xff000000u ? (_Float16) d : (_Float16) __builtin_nanf("");
}
// x / d to the nearest (ties to even), -8 .. 7, plus 8; inv = 1 / d rounded.  y = x inv is within
// two units of the quotient, so x - y d is exact and one more step leaves 2^-45 of it before
// the last rounding.  That rounding never crosses or meets a border (k + 1/2) d that x does
// not lie on: the border has at most 15 significant bits, so x is a unit of its own from it at
// least, which in the quotient is half a unit and 2^-16 of it more.
__device__ __forceinline__ uint32_t kv_code(float x, float d, float inv) {
    const float y = x * inv;
    const float q = __builtin_fmaf(__builtin_fmaf(-y, d, x), inv, y);
    return (uint32_t) ((int) fminf(fmaxf(__builtin_rintf(q), -8.0f), 7.0f) + 8);
}

// the rows' places: cell (for head 0, -1: passed over) and token in it
__device__ __forceinline__ void kv_places(const KvRowsArgs& a, int64_t r0, int64_t* s_cell, int* s_tok) {
    const int t = threadIdx.x;
    if (t < KV_ROWS) {
        const int64_t slot = r0 + t < a.T ? a.slot[r0 + t] : -1;
        const bool bad = slot >= 0 && slot >> a.c.page_shift >= a.c.n_pages;
        if (bad && blockIdx.y == 0 && blockIdx.z == 0) atomicOr(a.status, QWMOE_STATUS_BAD_SLOT);
        s_cell[t] = slot < 0 || bad ? -1 : a.c.cell(slot);
        s_tok[t] = (int) (slot & 31);
    }
}

template <int D, int PB, int TYPE>
__global__ void __launch_bounds__(256) k_kv_store(KvRowsArgs a) {
    constexpr int NB = D / 32, N = KV_ROWS * PB * 8 / 256, B = KV_ROWS * PB / 16;   // pieces of four dims, bytes of a value per lane
    __shared__ int64_t s_cell[KV_ROWS];
    __shared__ int s_tok[KV_ROWS];
    __shared__ uint32_t s_val[KV_ROWS][PB * 4 + 1];          // dword 4 b + l: byte j: dims 32 b + 4 l + j and 16 on
    const int64_t r0 = (int64_t) blockIdx.x * KV_ROWS;
    const int tid = threadIdx.x, hd = blockIdx.y >> 1, value = blockIdx.y & 1, b0 = blockIdx.z * PB;
    const int n_rows = (int) min((int64_t) KV_ROWS, a.T - r0);
    const size_t nb1 = value ? a.v_nb1 : a.k_nb1;
    const char* src = (const char*) (value ? a.v : a.k) + r0 * nb1 + ((size_t) hd * D + 32 * b0) * (TYPE == KV_F32 ? 4 : 2);
    float x[N][4];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int e = n * 256 + tid, r = e / (8 * PB);
        for (int j = 0; j < 4; ++j) x[n][j] = 0.0f;
        if (r < n_rows) kv_get4<TYPE>(src + r * nb1, e % (8 * PB), x[n]);
    }
    kv_places(a, r0, s_cell, s_tok);
    __syncthreads();
    uint8_t* base = a.c.data + hd * a.c.head_bytes() + (value ? 18 * D : 0);
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int e = n * 256 + tid, r = e / (8 * PB), b = e / 8 % PB, l = e & 7;
        uint32_t top = 0;
        for (int j = 0; j < 4; ++j) top = max(top, kv_rank(x[n][j]));
        const _Float16 d = kv_scale(kv_top8(top));
        const bool some = __builtin_fabsf((float) d) > 0.0f;   // (not 0 nor a NaN)
        const float inv = some ? 1.0f / (float) d : 0.0f;
        uint32_t key = 0, val = 0;   // this lane's four codes: nibbles of the key dword; one per byte
        for (int j = 0; j < 4; ++j) {
            const uint32_t c = some ? kv_code(x[n][j], (float) d, inv) : 8;
            key |= c << (4 * (j / 2 + 4 * (j & 1)));
            val |= c << (8 * j);
        }
        const int64_t cell = s_cell[r];
        const int tok = s_tok[r], tt = tok & 15, u = tok >> 4;
        if (value) {
            val |= kv_dpp<0x104>(val) << 4;   // (lanes 0 .. 3: the dims 16 further on in the high nibbles)
            if (l < 4) s_val[r][4 * b + l] = val;
        } else {
            key |= kv_dpp<0xB1>(key) << 8;   // (even lanes: dims 8 q + 4 .. in the upper bytes' nibbles)
            if (!(l & 1) && cell >= 0) ((uint32_t*) (base + cell))[((16 * u + tt) * 4 + l / 2) * NB + b0 + b] = key;
        }
        if (l == 0 && cell >= 0) ((_Float16*) (base + cell + 16 * D))[((4 * u + (tt >> 2)) * NB + b0 + b) * 4 + (tt & 3)] = d;
    }
    if (!value) return;
    __syncthreads();
    const int r = tid & (KV_ROWS - 1);
    const int64_t cell = s_cell[r];
    if (cell < 0) return;
    const int tok = s_tok[r], tt = tok & 15, u = tok >> 4;
    uint8_t* to = base + cell + ((tt >> 2) * 4 + u) * 4 + (tt & 3);
#pragma unroll
    for (int n = 0; n < B; ++n) {
        const int e = n * (256 / KV_ROWS) + tid / KV_ROWS, b = 2 * (e >> 5) + (e & 1), j = e >> 1 & 15;   // (two blocks' bytes lie in one line)
        to[((((b0 / 2 + (b >> 1)) * 16 + j) * 8 + (b & 1)) * 2) * 4] = (uint8_t) (s_val[r][4 * b + (j >> 2)] >> (8 * (j & 3)));
    }
}

template <int D, int PB, int TYPE>
__global__ void __launch_bounds__(256) k_kv_load(KvRowsArgs a) {
    constexpr int NB = D / 32, N = KV_ROWS * PB * 8 / 256, B = KV_ROWS * PB / 16;
    __shared__ int64_t s_cell[KV_ROWS];
    __shared__ int s_tok[KV_ROWS];
    __shared__ uint32_t s_val[KV_ROWS][PB * 4 + 1];
    const int64_t r0 = (int64_t) blockIdx.x * KV_ROWS;
    const int tid = threadIdx.x, hd = blockIdx.y >> 1, value = blockIdx.y & 1, b0 = blockIdx.z * PB;
    kv_places(a, r0, s_cell, s_tok);
    __syncthreads();
    const uint8_t* base = a.c.data + hd * a.c.head_bytes() + (value ? 18 * D : 0);
    float d[N];
    uint32_t code[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int e = n * 256 + tid, r = e / (8 * PB), b = e / 8 % PB, l = e & 7;
        const int64_t cell = s_cell[r];
        const int tok = s_tok[r], tt = tok & 15, u = tok >> 4;
        if (cell >= 0) {
            d[n] = (float) ((const _Float16*) (base + cell + 16 * D))[((4 * u + (tt >> 2)) * NB + b0 + b) * 4 + (tt & 3)];
            if (!value) code[n] = ((const uint32_t*) (base + cell))[((16 * u + tt) * 4 + l / 2) * NB + b0 + b];
        }
    }
    if (value) {
        const int r = tid & (KV_ROWS - 1);
        const int64_t cell = s_cell[r];
        const int tok = s_tok[r], tt = tok & 15, u = tok >> 4;
        const uint8_t* from = base + cell + ((tt >> 2) * 4 + u) * 4 + (tt & 3);
        uint8_t c[B];
#pragma unroll
        for (int n = 0; n < B; ++n) {
            const int e = n * (256 / KV_ROWS) + tid / KV_ROWS, b = 2 * (e >> 5) + (e & 1), j = e >> 1 & 15;
            if (cell >= 0) c[n] = from[((((b0 / 2 + (b >> 1)) * 16 + j) * 8 + (b & 1)) * 2) * 4];
        }
#pragma unroll
        for (int n = 0; n < B; ++n) {
            const int e = n * (256 / KV_ROWS) + tid / KV_ROWS, b = 2 * (e >> 5) + (e & 1), j = e >> 1 & 15;
            if (cell >= 0) ((uint8_t*) s_val[r])[16 * b + j] = c[n];
        }
        __syncthreads();
    }
    const size_t nb1 = value ? a.v_nb1 : a.k_nb1;
    char* dst = (char*) (value ? a.vo : a.ko) + r0 * nb1 + ((size_t) hd * D + 32 * b0) * (TYPE == KV_F32 ? 4 : 2);
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int e = n * 256 + tid, r = e / (8 * PB), b = e / 8 % PB, l = e & 7;
        if (s_cell[r] < 0) continue;
        float x[4];
        if (value) {
            const uint32_t c = s_val[r][4 * b + (l & 3)] >> (l & 4);
            for (int j = 0; j < 4; ++j) x[j] = d[n] * (float) ((int) (c >> (8 * j) & 15) - 8);
        } else {
            const uint32_t c = code[n] >> (8 * (l & 1));
            for (int j = 0; j < 4; ++j) x[j] = d[n] * (float) ((int) (c >> (4 * (j / 2 + 4 * (j & 1))) & 15) - 8);
        }
        kv_put4<TYPE>(dst + r * nb1, e % (8 * PB), x);
    }
}

int done() { return hipGetLastError() == hipSuccess ? 0 : -3; }

template <int D, int PB, int TYPE>
int launch_rows(const KvRowsArgs& a, bool load, hipStream_t st) {
    const int64_t tiles = (a.T + KV_ROWS - 1) / KV_ROWS;
    if (tiles > 0x7fffffff || 2 * a.c.n_head_kv > 65535) return -2;
    if (tiles == 0) return 0;
    const dim3 g((unsigned) tiles, (unsigned) (2 * a.c.n_head_kv), D / 32 / PB), b(256);
    if (load) hipLaunchKernelGGL((k_kv_load<D, PB, TYPE>), g, b, 0, st, a);
    else hipLaunchKernelGGL((k_kv_store<D, PB, TYPE>), g, b, 0, st, a);
    return done();
}
template <int D, int PB>
int launch_rows(const KvRowsArgs& a, bool load, hipStream_t st) {
    if (a.type == KV_F32) return launch_rows<D, PB, KV_F32>(a, load, st);
    if (a.type == KV_F16) return launch_rows<D, PB, KV_F16>(a, load, st);
    return launch_rows<D, PB, KV_BF16>(a, load, st);
}

// Whole heads per workgroup where that makes 1024 workgroups or more, else two blocks (the
// least whose value bytes fill a line): 77 rows of two heads of 256 in f16 4.8 us whole, 3.3
// by two blocks; 24 f32 rows of four heads of 128 in 3.4 and 2.9; 20000 of them out 20.3 and 22.6.
template <int D>
int launch_rows(const KvRowsArgs& a, bool load, hipStream_t st) {
    const bool whole = (a.T + KV_ROWS - 1) / KV_ROWS * 2 * a.c.n_head_kv >= 1024;
    return whole ? launch_rows<D, D / 32>(a, load, st) : launch_rows<D, 2>(a, load, st);
}
int launch_rows(const KvRowsArgs& a, bool load, hipStream_t st) {
    return a.c.D == 64 ? launch_rows<64>(a, load, st) : a.c.D == 128 ? launch_rows<128>(a, load, st) : launch_rows<256>(a, load, st);
}

}  // namespace

int launch_kv_plan(const KvPlanArgs& a, hipStream_t st) {
    if (a.S > KV_MAX_SEQ || a.T >= (int64_t(1) << 31)) return -2;
    const int64_t items = std::max<int64_t>(a.T, (int64_t) a.S * 64);
    const unsigned blocks = (unsigned) std::min<int64_t>((items + 255) / 256, 256);
    hipLaunchKernelGGL(k_kv_plan, dim3(std::max(blocks, 1u)), dim3(256), (size_t) 12 * (a.S + 1), st, a);
    return done();
}

int launch_kv_q4_store(const KvRowsArgs& a, hipStream_t st) { return launch_rows(a, false, st); }
int launch_kv_q4_load(const KvRowsArgs& a, hipStream_t st) { return launch_rows(a, true, st); }

}  // namespace qw
