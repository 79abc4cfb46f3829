// attn_q4.hip -- causal attention of a batch of requests over the paged 4-bit cache
// (layout in qw_kv_q4.hpp): row (token t of n, query head h) of request i sees its keys
// 0 .. len - n + t,
//   o = sum_j softmax_j(scale q . k_j) v_j.
//
// Requests of few rows (decode steps, drafts) are k_attn_q4's, requests of many (chunks of a prompt) are
// k_attn_q4_rows', which has its own notes.  Both form f16 operands of v_mfma_f32_16x16x32_f16 in
// registers: a code masked out of its dword is the f16 subnormal c 2^-24 (or, a nibble further on, c 2^-20), for
// two codes at once, and one packed multiply-add makes that (c - 8) 2^-9, exactly: nine
// instructions for eight operands.  (The subnormals themselves multiply too, but the
// products' sum then keeps 16 bits only.)
//
// Few rows: block scales are applied in fp32 around the products, so the cache's values enter
// unrounded:
//   scores   S^T = K Q^T, 16 keys x 16 rows, 32 dims (one block) a product; each block's
//            product is scaled by d_k of (key, block) as it is added;
//   values   O^T = V^T P^T, 16 dims x 16 rows, 32 keys a product, P's entries times d_v of (key,
//            block) and rounded to f16.
// The scores of a product lie in D as the next product's B operand wants them: lane l
// has row l % 16 and keys 4 (l / 16) + i of each 16, the order in which the cache keeps
// the value bytes.
//
// f32 rows are two f16 parts each, in two of a tile's columns: rows take columns
// 0 .. 7 with their high parts and 8 .. 15 with their low parts (q) and so do the
// weights; scores and outputs are the sums of both columns.  A decode step's eight
// query heads of a kv head then fill the tile that they would half leave empty.  q is scaled
// by a power of two to f16's upper range first, the weights by the running offset.
//
// The softmax's running maximum moves only when a weight would leave f16's range:
// weights are 2^(s - off), off = M + E - 4 with M the row's maximum and 2^E a bound of
// the value scales when it was last set, and it is set anew when some weight passes 2^12
// or some scale 2^E.  Otherwise a cell costs no exchange between lanes and no rescaling.
//
// A workgroup takes a request's rows (R = n_head / n_head_kv per token), one kv head and one
// split of the keys.  Its eight waves share out 16-column tiles of the rows, and waves of the
// same tile share out the cells; their sums meet in LDS, the splits' in a second launch.  Each
// wave copies its next cells straight into its own ring in LDS (no registers, no barrier: a wave
// waits for its own copies only), and the rings take what LDS there is: a workgroup to a CU.
//
// What bounds it: a long context reads its cells at the card's rate (one row of 131072 keys, four kv heads of 128,
// 75 MB: 24.0 us, about 4 of them before the first cell is there, and 4.4 for the join; a large sum reads 3.9 TB/s
// here); shorter ones wait for a chain of loads, lengths -> pages -> cells, and for each wave's 400 vector instructions
// a cell: one row of 700 keys 11.3 us, of which an empty kernel is 1.4; 24 requests of dozens to 8000 keys, 16 MB,
// 11.5 + 4.0; eight requests' five rows of up to 3000 keys at D = 256 16.6 + 6.3.  Against it: cells loaded into
// registers instead of the rings 35 us for the long context, 14.9 for the 700 keys; sixteen waves a workgroup, with
// half the registers each, slower.
#include <algorithm>
#include <type_traits>

#include "../../include/qwmoe.h"
#include "qw_kv_q4.hpp"
#include "qw_mfma.hpp"

namespace qw {

namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b4 __attribute__((ext_vector_type(4)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

constexpr float NO_KEY = -3.0e38f;   // M and off of a row that has seen no key yet

__device__ __forceinline__ void q4_put4(void* p, int type, int64_t i, f4 v) {
    if (type == KV_F32) *(f4*) ((float*) p + i) = v;
    else if (type == KV_F16) *(h4*) ((_Float16*) p + i) = __builtin_convertvector(v, h4);
    else *(b4*) ((__bf16*) p + i) = __builtin_convertvector(v, b4);
}

__device__ __forceinline__ void q4_put2(void* p, int type, int i, float x, float y) {
    if (type == KV_F32) *(float2*) ((float*) p + i) = float2{x, y};
    else if (type == KV_F16) *(h2*) ((_Float16*) p + i) = h2{(_Float16) x, (_Float16) y};
    else *(b2*) ((__bf16*) p + i) = b2{(__bf16) x, (__bf16) y};
}

__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// A request as the call gives it.
struct Q4Seq {
    int i, n, len;     // request, its new tokens, its keys (0: rows of zeros)
    int row0;          // its first token row
};
__device__ __forceinline__ bool q4_request(const AttnQ4Args& a, int i, Q4Seq& s) {
    s.i = i;
    s.row0 = a.seq_start[i];
    const int64_t end = a.seq_start[i + 1];
    s.len = a.seq_len[i];
    s.n = (int) (end - s.row0);
    return s.row0 >= 0 && end > s.row0 && end <= a.T;
}
// The last request whose key(first token row, number) is at most `want` (keys ascend).  Called
// by whole waves: 64 candidates at a time, whose rows and lengths come with the same loads.
template <typename F>
__device__ __forceinline__ bool q4_find(const AttnQ4Args& a, int lane, int64_t want, F key, Q4Seq& s) {
    int lo = 0, step = (a.S + 63) / 64;
    for (;;) {
        const int i = min(lo + lane * step, a.S - 1);
        const int t0 = a.seq_start[i], t1 = a.seq_start[i + 1], len = a.seq_len[i];
        const uint64_t m = __ballot(lo + lane * step < a.S && key(t0, i) <= want);
        if (m == 0) return false;
        const int at = 63 - __builtin_clzll(m);
        lo += at * step;
        if (step == 1) {
            s.i = uni(lo);
            s.row0 = __builtin_amdgcn_readlane(t0, at);
            const int64_t end = __builtin_amdgcn_readlane(t1, at);
            s.n = (int) (end - s.row0);
            s.len = __builtin_amdgcn_readlane(len, at);
            return s.row0 >= 0 && end > s.row0 && end <= a.T;
        }
        step = (step + 63) / 64;
    }
}
// Whether the request's lengths fit the call.
__device__ __forceinline__ bool q4_fits(const AttnQ4Args& a, const Q4Seq& s) {
    return s.len >= 0 && s.len <= a.max_len && s.n <= a.max_new;
}

// A cell's copy into LDS: instructions of 64 x 16 bytes, the rest of 64 x 4.
template <int D>
struct Q4Copy {
    static constexpr int BYTES = 36 * D, WIDE = BYTES / 1024, INSTR = WIDE + BYTES % 1024 / 256;
    static __device__ __forceinline__ void issue(const uint8_t* cell, uint8_t* slot, int l) {
        const i32x4 r = rsrc_words(cell, BYTES);
        const i32x4 rs = i32x4{uni(r.x), uni(r.y), uni(r.z), uni(r.w)};
        uint32_t lb = (uint32_t) uni((int) (uint32_t) (uintptr_t) slot);
        asm volatile("s_waitcnt lgkmcnt(0)" : "+s"(lb)::"memory");   // (the slot's last reads are done)
#pragma unroll
        for (int j = 0; j < WIDE; ++j) dma_b128(rs, lb + 1024u * j, (uint32_t) (16 * l + 1024 * j), 0u);
#pragma unroll
        for (int j = 0; j < INSTR - WIDE; ++j) dma_b32(rs, lb + 1024u * WIDE + 256u * j, (uint32_t) (4 * l + 1024 * WIDE + 256 * j), 0u);
    }
};

__device__ __forceinline__ float half_of(uint32_t w, int hi) {
    h2 x;
    __builtin_memcpy(&x, &w, 4);
    return (float) x[hi];
}
// v less the low or high half of w, in one instruction; or plus s times it
template <int HIGH>
__device__ __forceinline__ float less_half(float v, uint32_t w) {
    float r;
    if constexpr (HIGH) asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(w), "v"(v));
    else asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(w), "v"(v));
    return r;
}
template <int HIGH>
__device__ __forceinline__ float plus_half(float v, uint32_t w, float s) {
    float r;
    if constexpr (HIGH) asm("v_fma_mix_f32 %0, %1, %2, %3 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(w), "v"(s), "v"(v));
    else asm("v_fma_mix_f32 %0, %1, %2, %3 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(w), "v"(s), "v"(v));
    return r;
}
__device__ __forceinline__ uint32_t word_of(_Float16 lo, _Float16 hi) {
    const h2 x = {lo, hi};
    uint32_t w;
    __builtin_memcpy(&w, &x, 4);
    return w;
}
__device__ __forceinline__ h8 as_h8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    const u32x4 w = {a, b, c, d};
    h8 r;
    __builtin_memcpy(&r, &w, 16);
    return r;
}
// The codes in the low (shift 0) or high (1) nibbles of bytes 0 and 2, less 8, times 2^-9.
template <int HIGH>
__device__ __forceinline__ uint32_t codes(uint32_t w) {
    constexpr _Float16 up = HIGH ? 2048.0f : 32768.0f, eight = 0x1p-6f;
    w &= HIGH ? 0x00f000f0u : 0x000f000fu;
    h2 x;
    __builtin_memcpy(&x, &w, 4);
    x = __builtin_elementwise_fma(x, h2{up, up}, h2{-eight, -eight});
    __builtin_memcpy(&w, &x, 4);
    return w;
}

// The values of lanes l ^ 16 and l ^ 32 join this lane's: all four groups of 16 then agree.
template <typename F>
__device__ __forceinline__ float over_groups(float v, F join) {
    auto a = __builtin_amdgcn_permlane16_swap(fbits(v), fbits(v), false, false);
    v = join(bitsf(a[0]), bitsf(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(fbits(v), fbits(v), false, false);
    return join(bitsf(b[0]), bitsf(b[1]));
}
__device__ __forceinline__ float max_over_16(float v) {
    v = fmaxf(v, dpp_f<0x121>(v));   // row_ror 1, 2, 4, 8
    v = fmaxf(v, dpp_f<0x122>(v));
    v = fmaxf(v, dpp_f<0x124>(v));
    return fmaxf(v, dpp_f<0x128>(v));
}
__device__ __forceinline__ float max_over_groups(float v) {
    return over_groups(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float sum_over_groups(float v) {
    return over_groups(v, [](float a, float b) { return a + b; });
}
// The largest of all lanes' values below 2^16.
__device__ __forceinline__ int max_of_wave(int v) {
    v = max(v, dpp_i<0x121>(v));   // row_ror 1, 2, 4, 8
    v = max(v, dpp_i<0x122>(v));
    v = max(v, dpp_i<0x124>(v));
    v = max(v, dpp_i<0x128>(v));
    return max(max(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
               max(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}

// (lane l ^ 8 of the same 16)
__device__ __forceinline__ float other_part(float v) { return dpp_f<0x128>(v); }   // row_ror:8

// Waves of a workgroup: two to a SIMD (more have too few registers, and each brings its own q and sums).  Cells of a wave in flight or in
// use: as many as LDS holds.
constexpr int q4_waves(int D) { return 8; }
constexpr int q4_ring(int D) { return D == 64 ? 4 : D == 128 ? 3 : 2; }
constexpr int Q4_TILES = 8;   // of a request that k_attn_q4 takes

// A row's q (NS f16 parts; lane l has dims 8 (l / 16) .. of each block, f32 rows' low parts in
// columns 8 .. 15): its dwords, then the parts, scaled by a power of two into f16's upper range.
// parts() returns the scores' factor: scale log2(e) over that power.
template <int D, int NS>
struct Q4Row {
    static constexpr int NB = D / 32;
    u32x4 x[NB][NS];
    __device__ __forceinline__ void load(const AttnQ4Args& a, int tok, int h, int l) {
        const char* src = (const char*) a.q + (int64_t) tok * a.q_nb1 + (uint32_t) (h * D + 8 * (l >> 4)) * (2 * NS);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < NS; ++e) x[b][e] = *(const u32x4*) (src + 64 * NS * b + 16 * e);
    }
    __device__ __forceinline__ float parts(const AttnQ4Args& a, bool ok, h8 (&q)[NS][NB]) const {
        const bool f16 = a.type == KV_F16;
        auto value = [&](int b, int j) {
            if constexpr (NS == 2) return bitsf(x[b][j / 4][j % 4]);
            const uint32_t word = x[b][0][j / 2];
            return f16 ? half_of(word, j & 1) : bitsf(j & 1 ? word & 0xffff0000u : word << 16);
        };
        float big = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int j = 0; j < 8; ++j) big = fmaxf(big, __builtin_fabsf(value(b, j)));
        big = max_over_groups(big);
        // 2^ex <= big < 2^(ex + 1): q 2^(14 - ex)
        const int ex = min(max((int) (fbits(big) >> 23) - 127, -60), 127);
        const float up = bitsf((uint32_t) (127 + 14 - ex) << 23);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            uint32_t w[NS][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float y0 = value(b, 2 * j) * up, y1 = value(b, 2 * j + 1) * up;
                w[0][j] = word_of((_Float16) y0, (_Float16) y1);
                if (NS == 2) w[NS - 1][j] = word_of((_Float16) (y0 - half_of(w[0][j], 0)), (_Float16) (y1 - half_of(w[0][j], 1)));
            }
#pragma unroll
            for (int e = 0; e < NS; ++e) q[e][b] = ok ? as_h8(w[e][0], w[e][1], w[e][2], w[e][3]) : as_h8(0, 0, 0, 0);
        }
        return a.scale * bitsf((uint32_t) (127 - 14 + ex) << 23);
    }
};

// NS f16 parts per row (f32 rows: two).
template <int D, int NS>
__global__ void __launch_bounds__(64 * q4_waves(D)) __attribute__((amdgpu_waves_per_eu(q4_waves(D) / 4, q4_waves(D) / 4))) k_attn_q4(AttnQ4Args a) {
    constexpr int NB = D / 32, RC = 16 / NS, W = q4_waves(D), N = q4_ring(D), I = Q4Copy<D>::INSTR, SLOT = Q4Copy<D>::BYTES;
    constexpr int LD = D + 4;                                   // floats of a row where the waves' sums meet
    __shared__ __align__(16) uint8_t s_ring[W * (N * SLOT > RC * LD * 4 ? N * SLOT : RC * LD * 4)];
    __shared__ float2 s_ol[W][RC];                              // offset and sum of weights
    constexpr int LQ = D + 8;                                   // halves of a row's q
    __shared__ float s_qs[RC * Q4_TILES];
    const int tid = threadIdx.x, l = tid & 63, m = l & 15, g = l >> 4;
    const int w = uni(tid >> 6);
    const int R = a.group, hd = blockIdx.y;
    auto by_R = [&](int r) { return R == 1 ? r : (int) __umulhi((unsigned) r, a.group_inv); };   // r / R for 0 <= r < 2^16
    const int cpp = a.c.page_shift - 5;                         // log2 of a page's cells
    Q4Seq s;
    int z, unit;                                                // the split: of the request, and where its sums go
    int64_t per = a.cells;
    if (a.units) {
        // As many cells to a split that the requests' splits are `units` or fewer: a lane has a request.
        const int i = min(l, a.S - 1), t0 = a.seq_start[i], t1 = a.seq_start[i + 1], n = t1 - t0;
        s.len = a.seq_len[i];
        s.n = n;
        const bool mine = l < a.S && t0 >= 0 && t1 > t0 && t1 <= a.T && (n > a.max_new || (int64_t) n * R <= Q4_TILES * RC);
        const unsigned c = !mine ? 0 : q4_fits(a, s) ? (unsigned) max((s.len + 31) >> 5, 1) : 1;
        auto splits = [&](unsigned p) { return (c + p - 1) / p; };
        auto sum = [&](unsigned v) { return (unsigned) __builtin_amdgcn_readlane((int) kv_wave_incl(v), 63); };
        const unsigned all = sum(c), units = (unsigned) a.units, spare = units - (unsigned) a.S;
        // (splits of p cells are at most all / p + S)
        unsigned lo = max((all - 1) / units + 1, (unsigned) a.least), hi = max((all - 1) / spare + 1, lo);
        while (lo < hi) {
            const unsigned p = (lo + hi) / 2;
            if (sum(splits(p)) <= units) hi = p;
            else lo = p + 1;
        }
        const unsigned mine_n = splits(lo), end = kv_wave_incl(mine_n);
        const uint64_t has = __ballot(blockIdx.x >= end - mine_n && blockIdx.x < end);
        if (has == 0) return;
        const int at = __builtin_ctzll(has);
        s = Q4Seq{at, __builtin_amdgcn_readlane(n, at), __builtin_amdgcn_readlane(s.len, at), __builtin_amdgcn_readlane(t0, at)};
        const int before = __builtin_amdgcn_readlane((int) (end - mine_n), at);
        per = lo;
        unit = blockIdx.x;
        z = unit - before;
        if (z == 0 && hd == 0 && tid == 0) a.first[at] = int2{before, (int) lo};
    } else {
        s.i = blockIdx.x;
        z = blockIdx.z;
        unit = z * a.S + s.i;
    }
    // pages of the split's cells, 64 at a time, one per lane (entries behind the request's are read, not used: they
    // come in with its lengths)
    const int32_t* pages = a.table + (int64_t) s.i * a.W;
    const int zc = (int) min(z * per, (int64_t) 1 << 30);
    int pg_at = zc >> cpp, pg = pages[min((int64_t) pg_at + l, a.W - 1)];
    if (!a.units && !q4_request(a, s.i, s)) return;
    const int rows = (int) min((int64_t) s.n * R, (int64_t) 1 << 30);
    if (s.n > a.max_new) {                                      // however many rows: zeros
        if (z > 0) return;
        if (tid == 0) atomicOr(a.status, QWMOE_STATUS_BAD_SEQ);
        for (int64_t e = tid; e < (int64_t) s.n * R * (D / 4); e += 64 * W) {
            const int64_t row = e / (D / 4);
            q4_put4((char*) a.out + (s.row0 + row / R) * a.out_nb1, a.type, (hd * R + row % R) * D + 4 * (e % (D / 4)), f4{0.0f, 0.0f, 0.0f, 0.0f});
        }
        return;
    }
    if (rows > Q4_TILES * RC) return;                           // (k_attn_q4_rows')
    int len = s.len;
    if (!q4_fits(a, s)) {
        len = 0;
        if (tid == 0) atomicOr(a.status, QWMOE_STATUS_BAD_SEQ);
    }
    // the waves of the workgroup: 2^tshift tiles of rows, 2^cshift waves each
    const int tshift = rows <= RC ? 0 : rows <= 2 * RC ? 1 : rows <= 4 * RC ? 2 : 3;
    const int cshift = 3 - tshift;
    const int r0 = (w & ((1 << tshift) - 1)) * RC;              // the wave's first row
    const int wrows = max(min(rows - r0, RC), 0);
    const int back = len - s.n;                                 // a row of token t sees keys .. back + t
    const int last = wrows ? back + by_R(r0 + wrows - 1) : -1;  // the last key some row of the wave sees
    const int every = back + by_R(r0);                          // keys up to here are seen by all of its rows
    const int cells = last < 0 ? 0 : (last >> 5) + 1;
    if (z > 0 && zc > (len - 1) >> 5) return;                   // (z = 0 writes the rows without keys)
    const int c0 = min(zc + (w >> tshift), cells);              // its cells: c0, c0 + 2^cshift ..
    const int c1 = (int) min(zc + per, (int64_t) cells);

    // this lane's row
    const int r = r0 + (m & (RC - 1));
    const bool ok = r < rows;
    const int lim = ok ? back + by_R(r) : -1;                   // the last key it sees
    const uint8_t* head = a.c.data + hd * a.c.head_bytes();
    const int64_t page_bytes = a.c.page_bytes();
    uint8_t* ring = s_ring + w * SLOT;                          // [slot][wave]
    uint32_t bad = 0;                                           // bit k: the cell in slot k has no page
    auto issue = [&](int c, int slot) __attribute__((always_inline)) {
        if ((c >> cpp) - pg_at >= 64) {
            pg_at = c >> cpp;
            pg = pages[min((int64_t) pg_at + l, a.W - 1)];
        }
        const int page = __builtin_amdgcn_readlane(pg, (c >> cpp) - pg_at);
        const bool ok = page >= 0 && page < a.c.n_pages;
        if (!ok && l == 0) atomicOr(a.status, QWMOE_STATUS_BAD_SLOT);
        bad = ok ? bad & ~(1u << slot) : bad | 1u << slot;
        Q4Copy<D>::issue(head + (ok ? page : 0) * page_bytes + (c & ((1 << cpp) - 1)) * (36 * D), ring + slot * (W * SLOT), l);
    };
#pragma unroll
    for (int k = 0; k < N - 1; ++k)
        if (c0 + (k << cshift) < c1) issue(c0 + (k << cshift), k);

    // q, a row per wave in turn: scaled by a power of two into f16's upper range, its parts to LDS (where the
    // rings' last slots, still unused, are)
    _Float16* s_q = (_Float16*) (s_ring + (N - 1) * W * SLOT);
    static_assert(NS * RC * Q4_TILES * LQ * 2 <= W * SLOT, "q fits the last slots");
    constexpr int E4 = 4, EV = D / 64;                          // rows of a wave at a time, their values of a lane
    for (int i0 = w; i0 < (RC << tshift); i0 += E4 * W) {
        uint8_t raw[E4][EV * 2 * NS];
#pragma unroll
        for (int j = 0; j < E4; ++j) {                          // (rows behind the last one: the last one's)
            const int i = min(i0 + j * W, rows - 1), t = by_R(i), h = hd * R + i - t * R;
            __builtin_memcpy(raw[j], __builtin_assume_aligned((const char*) a.q + (int64_t) (s.row0 + t) * a.q_nb1 + (h * D + EV * l) * (2 * NS),
                                                              EV * 2 * NS), EV * 2 * NS);
        }
#pragma unroll
        for (int j = 0; j < E4; ++j) {
            const int i = i0 + j * W;
            if (i >= (RC << tshift)) break;
            float x[EV], big = 0.0f;
#pragma unroll
            for (int e = 0; e < EV; ++e) {
                if constexpr (NS == 2) __builtin_memcpy(&x[e], raw[j] + 4 * e, 4);
                else {
                    uint16_t v;
                    __builtin_memcpy(&v, raw[j] + 2 * e, 2);
                    x[e] = a.type == KV_F16 ? (float) __builtin_bit_cast(_Float16, v) : bitsf((uint32_t) v << 16);
                }
                x[e] = i < rows ? x[e] : 0.0f;
                big = fmaxf(big, __builtin_fabsf(x[e]));
            }
            big = max_over_groups(max_over_16(big));
            // 2^ex <= big < 2^(ex + 1): q 2^(14 - ex)
            const int ex = min(max((int) (fbits(big) >> 23) - 127, -60), 127);
            const float up = bitsf((uint32_t) (127 + 14 - ex) << 23);
            _Float16* dst = s_q + i * LQ + EV * l;
#pragma unroll
            for (int e = 0; e < EV; ++e) {
                const float y = x[e] * up;
                const _Float16 hi = (_Float16) y;
                dst[e] = hi;
                if (NS == 2) dst[8 * Q4_TILES * LQ + e] = (_Float16) (y - (float) hi);
            }
            if (l == 0) s_qs[i] = 512.0f * a.scale * bitsf((uint32_t) (127 - 14 + ex) << 23);
        }
    }
    lds_barrier();   // (the cells' copies stay in flight)
    h8 q[NB];
    {
        const _Float16* src = s_q + ((NS == 2 && m >= RC ? 8 * Q4_TILES : 0) + r0 + (m & (RC - 1))) * LQ + 8 * g;
#pragma unroll
        for (int b = 0; b < NB; ++b) q[b] = *(const h8*) (src + 32 * b);
    }
    lds_barrier();
    const float qs = s_qs[r0 + (m & (RC - 1))];                 // the scores' factor: scale log2(e), 2^9 for the codes, q's power of two

    f4 o[2 * NB];                // O^T 2^-9: dims 16 tile + 4 g + i of the lane's row
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) o[i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    float off = NO_KEY, mx = NO_KEY, lsum = 0.0f;
    int E = -25;                 // the value scales so far are at most 2^E
    int Ebits = 0;               // 2^E as f16 bits

    const float less = m < RC ? 0.0f : -1.0f;                   // (lanes with low parts: what the high one leaves)
    int slot = 0;
    for (int c = c0; c < c1; c += 1 << cshift) {
        const int ahead = c + ((N - 1) << cshift);
        const bool gone = bad >> slot & 1;
        if (ahead < c1) {
            issue(ahead, slot == 0 ? N - 1 : slot - 1);
            vm_wait<(N - 1) * I>();
        } else if (N > 2 && c + ((N - 2) << cshift) < c1) vm_wait<(N > 2 ? N - 2 : 0) * I>();
        else if (N > 3 && c + ((N - 3) << cshift) < c1) vm_wait<(N > 3 ? N - 3 : 0) * I>();
        else vm_wait<0>();
        const uint8_t* cell = ring + slot * (W * SLOT);
        slot = slot == N - 1 ? 0 : slot + 1;
        uint32_t kc[2][NB], kd[2][NB][2], vc[NB][2], vd[2][NB][2], chk[(NB + 3) / 4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            __builtin_memcpy(kc[u], __builtin_assume_aligned(cell + ((16 * u + m) * 4 + g) * NB * 4, NB == 2 ? 8 : 16), 4 * NB);
            __builtin_memcpy(kd[u], __builtin_assume_aligned(cell + 16 * D + (4 * u + g) * NB * 8, 16), 8 * NB);
        }
        if constexpr (NB == 2) chk[0] = *(const uint16_t*) (cell + 34 * D + 2 * l);
        else __builtin_memcpy(chk, __builtin_assume_aligned(cell + 34 * D + NB * l, NB), NB);
#pragma unroll
        for (int u = 0; u < 2; ++u) __builtin_memcpy(vd[u], __builtin_assume_aligned(cell + 34 * D + (4 * u + g) * NB * 8, 16), 8 * NB);
#pragma unroll
        for (int b = 0; b < NB; b += 2)
            __builtin_memcpy(vc[b], __builtin_assume_aligned(cell + 18 * D + (((b / 2) * 16 + m) * 4 + g) * 16, 16), 16);
        const bool masked = 32 * c + 31 > every || gone;        // some row does not see some key of the cell
        const int key0 = 32 * c + 4 * g, see = gone ? -1 : lim; // key i of half u: key0 + 16 u + i
        f4 sc[2] = {f4{0.0f, 0.0f, 0.0f, 0.0f}, f4{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const uint32_t c4 = kc[u][b], d4 = c4 >> 8;
                const h8 ka = as_h8(codes<0>(c4), codes<1>(c4), codes<0>(d4), codes<1>(d4));
                const f4 p = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, q[b], f4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) sc[u][i] = __builtin_fmaf(p[i], half_of(kd[u][b][i / 2], i & 1), sc[u][i]);
            }
        // the largest value scale of the request's keys, as f16 bits (NaNs count as 0), from the lane's share
        int top = 0;
#pragma unroll
        for (int e = 0; e < NB / 2; ++e) {
            const int x = (int) (chk[e / 2] >> (16 * (e & 1))) & 0x7fff;
            const int at = l * (NB / 2) + e, key = 4 * (at / (4 * NB)) + at % 4;
            top = max(top, x > 0x7c00 || key > last - 32 * c ? 0 : x);
        }
        if (NS == 2)
#pragma unroll
            for (int i = 0; i < 8; ++i) sc[i / 4][i % 4] += other_part(sc[i / 4][i % 4]);
        if (masked)
#pragma unroll
            for (int i = 0; i < 8; ++i) sc[i / 4][i % 4] = key0 + 16 * (i / 4) + i % 4 <= see ? sc[i / 4][i % 4] : -INFINITY;
        float smax = sc[0][0];
#pragma unroll
        for (int i = 1; i < 8; ++i) smax = fmaxf(smax, sc[i / 4][i % 4]);
        if (__any(top > Ebits || __builtin_fmaf(smax, qs, -off) > 12.0f - (float) E)) {
            const int t = max_of_wave(top);
            if (t > Ebits) {   // the power of two above the largest scale (from 2^-14 on, f16's smallest normal number)
                E = max(t >> 10, 1) - 14;
                Ebits = (E + 15) << 10;
            }
            mx = fmaxf(mx, max_over_groups(smax) * qs);
            const float now = mx == NO_KEY ? NO_KEY : mx + (float) (E - 4), f = exp2_hw(off - now);
            off = now;
            lsum *= f;
#pragma unroll
            for (int i = 0; i < 2 * NB; ++i) o[i] *= f;
        }
        // weights, formed in place
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float p = exp2_hw(__builtin_fmaf(sc[i / 4][i % 4], qs, -off));
            sc[i / 4][i % 4] = p;
            lsum += p;
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const uint32_t x0 = vc[b][0], x1 = vc[b][1], y0 = x0 >> 8, y1 = x1 >> 8;
            const h8 va[2] = {as_h8(codes<0>(x0), codes<0>(y0), codes<0>(x1), codes<0>(y1)),
                              as_h8(codes<1>(x0), codes<1>(y0), codes<1>(x1), codes<1>(y1))};
            {
                uint32_t pw[4];   // keys i and i + 2 of each half
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int u = k / 2, i = k % 2;
                    const float p0 = sc[u][i], p1 = sc[u][i + 2];
                    const float d0 = half_of(vd[u][b][0], i), d1 = half_of(vd[u][b][1], i);
                    // (one fp32 rounding of the products whatever the compiler would make of them)
                    float w0 = __builtin_fmaf(p0, d0, 0.0f), w1 = __builtin_fmaf(p1, d1, 0.0f);
                    asm volatile("" : "+v"(w0), "+v"(w1));
                    uint32_t hi = word_of((_Float16) w0, (_Float16) w1);
                    if (NS == 2) hi = word_of((_Float16) plus_half<0>(w0, hi, less), (_Float16) plus_half<1>(w1, hi, less));
                    pw[k] = hi;
                }
                if (masked)   // (a masked key's scale may be a NaN)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int key = key0 + 16 * (k / 2) + k % 2;
                        pw[k] &= (key <= see ? 0xffffu : 0u) | (key + 2 <= see ? 0xffff0000u : 0u);
                    }
                const h8 pb = as_h8(pw[0], pw[1], pw[2], pw[3]);
#pragma unroll
                for (int k = 0; k < 2; ++k) o[2 * b + k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va[k], pb, o[2 * b + k], 0, 0, 0);
            }
        }
    }

    // the waves' sums meet in LDS
    lsum = sum_over_groups(lsum);
    if (l < RC) s_ol[w][l] = float2{off, lsum};
    if (NS == 2)
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] += other_part(o[i][j]);
    __syncthreads();   // (every wave is done with its ring)
    float* s_o = (float*) s_ring;
    if (m < RC)
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) *(f4*) (s_o + (w * RC + m) * LD + 16 * i + 4 * g) = o[i];
    const int tiles = 1 << tshift;
    __syncthreads();
    auto join = [&](auto ways_) __attribute__((always_inline)) {
        constexpr int ways = decltype(ways_)::value;
        for (int e = tid; e < rows * (D / 2); e += 64 * W) {
            const int row = e / (D / 2), dim = 2 * (e % (D / 2)), tile = row / RC, rr = row % RC;
            float2 ol[ways], part[ways];
#pragma unroll
            for (int k = 0; k < ways; ++k) {
                const int from = tile + tiles * k;
                ol[k] = s_ol[from][rr];
                part[k] = *(const float2*) (s_o + (from * RC + rr) * LD + dim);
            }
            float at = ol[0].x, sum = 0.0f;
#pragma unroll
            for (int k = 1; k < ways; ++k) at = fmaxf(at, ol[k].x);
            float2 v = float2{0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < ways; ++k) {
                const float f = exp2_hw(ol[k].x - at);
                v.x += part[k].x * f;
                v.y += part[k].y * f;
                sum += ol[k].y * f;
            }
            const int tok = by_R(row), hh = hd * R + row - tok * R, lastc = (back + tok) >> 5;
            if (lastc < per) {              // the row's keys are all in the first split
                if (z > 0) continue;
                const float inv = sum == 0.0f ? 0.0f : 512.0f / sum;
                q4_put2((char*) a.out + (int64_t) (s.row0 + tok) * a.out_nb1, a.type, hh * D + dim, v.x * inv, v.y * inv);
            } else if (zc <= lastc) {
                const int64_t p = ((int64_t) unit * a.tcap + tok) * a.n_head + hh;
                *(float2*) (a.part + p * D + dim) = float2{v.x * 512.0f, v.y * 512.0f};
                if (dim == 0) *(float2*) (a.stat + 2 * p) = float2{at, sum};
            }
        }
    };
    switch (cshift) {
        case 0: join(std::integral_constant<int, 1>()); break;
        case 1: join(std::integral_constant<int, 2>()); break;
        case 2: join(std::integral_constant<int, 4>()); break;
        default: join(std::integral_constant<int, 8>());
    }
}

// ---- many rows per request ------------------------------------------------------
//
// A workgroup of eight waves takes 16-column tiles of a request's rows and one kv head.  Here
// a cell serves many tiles, so its values are formed once, d (code - 8) itself, as matrix
// core operands in LDS: no scaling around the products then, and a weight enters once, not
// once per block.  The product of an 11-bit scale and a 4-bit code has 15 bits: f32 and f16
// rows take it exactly as two f16 parts (EXACT), bf16 rows as one, whose 2^-12 is far below
// their own rounding.  Scales are brought into f16's range by powers of two, 2^sk and 2^sv,
// that only fall, where some cell's largest scale asks for it (every wave looks at every
// scale, so all agree without exchange).
//
// f32 rows are two f16 parts in separate operands: of the four products of parts, low by low is left out
// (2^-24 of the whole, a step of fp32).
//
// D <= 128: four waves' rows, two tiles each, and two cells at a time, one per half of the waves,
// whose sums meet in LDS at the end; D = 256: eight waves' rows, a tile each, one cell at a time.
// Two buffers: the next step's operands are formed, and the one after's dwords loaded, while this
// one's are used; one barrier a step.  One of a SIMD's two waves forms while the other multiplies.
//
// What bounds it: the instructions around the products.  A wave's 64 keys take 96 products (f32 rows, D = 128: 1600
// clocks alone), about 130 vector instructions to form its share of the operands and 100 for two tiles' softmax, at 4 clocks
// and more each beside a product; measured 2.9 us a step where the products of both waves need 1.5.  A chunk of
// 512 tokens behind 1037 (32 heads on 4, D = 128): f32 49.5 us + 5.8 to join two splits, f16 43 + 5.2, bf16 37 + 5.2;
// one of 1024 bf16 tokens up to 4000 keys 109 us (58.8 Gflop, 540 Tflop/s).  Of a chunk's time about 12 us lie before
// the first product (lengths, pages, q) and behind the last (sums, output).  Tried and slower: four waves to a SIMD
// with a tile each (f32 63.8 us: spills), the next operands formed between this step's products in one wave (54.0),
// one tile a wave (58.8 unsplit).
//
// A NaN scale of a value is taken as 0 and its block set to NaN afterwards in the rows that
// see the key: 0 times NaN would reach those that do not.
// (16 x 16 tiles of a wave, halves of the workgroup: what 256 registers and 160 KiB of LDS hold)
constexpr int qr_tiles(int D) { return D == 256 ? 1 : 2; }
constexpr int qr_halves(int D) { return D == 256 ? 1 : 2; }

__device__ __forceinline__ uint32_t mul_h2(uint32_t a, uint32_t b) {
    h2 x, y;
    __builtin_memcpy(&x, &a, 4);
    __builtin_memcpy(&y, &b, 4);
    x = x * y;
    __builtin_memcpy(&a, &x, 4);
    return a;
}
// a b - c, rounded once
__device__ __forceinline__ uint32_t rest_h2(uint32_t a, uint32_t b, uint32_t c) {
    h2 x, y, v;
    __builtin_memcpy(&x, &a, 4);
    __builtin_memcpy(&y, &b, 4);
    __builtin_memcpy(&v, &c, 4);
    x = __builtin_elementwise_fma(x, y, -v);
    __builtin_memcpy(&a, &x, 4);
    return a;
}
__device__ __forceinline__ uint32_t pow2_h2(int e) {   // 2^e in both halves, -14 <= e <= 15
    const uint32_t x = (uint32_t) (e + 15) << 10;
    return x | x << 16;
}

template <int D, int NS, bool EXACT>
__global__ void __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) k_attn_q4_rows(AttnQ4Args a, int most) {
    constexpr int NB = D / 32, RC = 16, NC = qr_tiles(D), KH = qr_halves(D), RG = 8 / KH, RW = NC * RC, RB = RG * RW;
    constexpr int RN = 8 / KH, PF = 2 * NB / RN;                // waves that form a cell's operands, K (and V) operands of each
    constexpr int PARTS = EXACT ? 2 : 1, FR = 4 * NB;           // a cell: FR operands of 64 lanes x 16 bytes per part
    __shared__ __align__(16) uint8_t s_mem[2 * KH * PARTS * FR * 1024];
    __shared__ float s_off[4][NC][64], s_l[4][NC][64];
    const int tid = threadIdx.x, l = tid & 63, m = l & 15, g = l >> 4;
    const int w = uni(tid >> 6), rg = w % RG, kh = w / RG, role = w % RN;
    const unsigned R = (unsigned) a.n_head / (unsigned) a.c.n_head_kv;
    const int hd = blockIdx.y, z = blockIdx.z;
    Q4Seq s;
    if (!q4_find(a, l, blockIdx.x, [&](int t, int i) { return (int64_t) max(t, 0) * R / RB + i; }, s)) return;
    const int rows = (int) min((int64_t) s.n * R, (int64_t) 1 << 30);
    if (rows <= most || (most && s.n > a.max_new)) return;      // (k_attn_q4's)
    // the request's blocks, the last rows (the most keys) first
    const int blocks = (rows + RB - 1) / RB, at = blockIdx.x - (int) ((int64_t) s.row0 * R / RB + s.i);
    if (at >= blocks) return;
    const int base = (blocks - 1 - at) * RB;
    int len = s.len;
    if (!q4_fits(a, s)) {
        len = 0;
        if (tid == 0) atomicOr(a.status, QWMOE_STATUS_BAD_SEQ);
    }
    const int r0 = base + rg * RW, wrows = max(min(rows - r0, RW), 0), back = len - s.n;
    const int block_last = back + (int) ((unsigned) (min(rows, base + RB) - 1) / R);
    const int last = wrows ? back + (int) ((unsigned) (r0 + wrows - 1) / R) : -1;
    const int every = back + (int) ((unsigned) r0 / R);
    const int zc = (int) min((int64_t) z * a.row_cells, (int64_t) 1 << 30);
    if (z > 0 && zc > block_last >> 5) return;
    const int cend = block_last < 0 ? zc : (int) min(zc + a.row_cells, (int64_t) (block_last >> 5) + 1);   // cells zc .. cend - 1
    const int steps = (cend - zc + KH - 1) / KH;

    const int32_t* pages = a.table + (int64_t) s.i * a.W;
    const int cpp = a.c.page_shift - 5;
    const uint8_t* head = a.c.data + hd * a.c.head_bytes();
    const int64_t page_bytes = a.c.page_bytes();
    // pages of 64 cells at a time, one per lane
    int pg_at = zc, pg = zc + l < cend ? pages[(zc + l) >> cpp] : 0;
    // this lane's rows, asked for together with the first pages
    Q4Row<D, NS> qx[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        const int r = min(r0 + n * RC + m, rows - 1);
        qx[n].load(a, s.row0 + (int) ((unsigned) r / R), hd * (int) R + (int) ((unsigned) r % R), l);
    }
    auto check_pages = [&] {
        if (pg < 0 || pg >= a.c.n_pages) {
            atomicOr(a.status, QWMOE_STATUS_BAD_SLOT);
            pg = -1;
        }
    };
    // this wave's share of a step: one cell's dwords, and all of the step's scales
    uint32_t kc[PF], vc[2], vd[2][2], chk[KH][2][(NB + 3) / 4];
    uint16_t kd[PF];
    int page[KH];
    const int kf = role * PF, ku = kf / NB, kb = kf % NB;       // its K operands: half ku, blocks kb ..
    const int vb = role * PF / 2;                               // its V operands: block vb (with one operand: half role % 2)
    auto load = [&](int step) __attribute__((always_inline)) {
        const int c = zc + step * KH;
        if (c + KH - 1 - pg_at >= 64) {
            pg_at = c;
            pg = c + l < cend ? pages[(c + l) >> cpp] : 0;
            check_pages();
        }
#pragma unroll
        for (int k = 0; k < KH; ++k) {
            const int ck = min(c + k, cend - 1);
            page[k] = c + k < cend ? __builtin_amdgcn_readlane(pg, ck - pg_at) : -1;
            const uint8_t* cell = head + max(page[k], 0) * page_bytes + (ck & ((1 << cpp) - 1)) * (36 * D);
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if constexpr (NB == 2) chk[k][e][0] = *(const uint16_t*) (cell + (uint32_t) ((e ? 34 : 16) * D + 2 * l));
                else __builtin_memcpy(chk[k][e], cell + (uint32_t) ((e ? 34 : 16) * D + NB * l), NB);
            if (w / RN == k) {
                __builtin_memcpy(kc, cell + (uint32_t) ((((16 * ku + m) * 4 + g) * NB + kb) * 4), 4 * PF);
#pragma unroll
                for (int j = 0; j < PF; ++j)
                    kd[j] = *(const uint16_t*) (cell + (uint32_t) (16 * D + (((4 * ku + (m >> 2)) * NB + kb + j) * 4 + (m & 3)) * 2));
                __builtin_memcpy(vc, cell + (uint32_t) (18 * D + ((((vb >> 1) * 16 + m) * 4 + g) * 2 + (vb & 1)) * 8), 8);
#pragma unroll
                for (int u = 0; u < 2; ++u) __builtin_memcpy(vd[u], cell + (uint32_t) (34 * D + ((4 * u + g) * NB + vb) * 8), 8);
            }
        }
    };
    int sk = 15, sv = 15;                                       // of the operands formed last
    int nans = 0, gone = 0;                                     // bit k: cell k of it holds a NaN value scale; has no page
    auto operand = [&](int buf, int cellk, int part, int f) {
        return s_mem + ((((buf * KH + cellk) * PARTS + part) * FR + f) * 64 + l) * 16;
    };
    auto form = [&](int step, int buf) __attribute__((always_inline)) {
        const int c = zc + step * KH;
        // the powers of two: every scale below 2^15 after them.  One comparison per kind says that they stand (keys
        // behind the request's may fail it for nothing)
        nans = gone = 0;
        u16x2 raw[2] = {u16x2{0, 0}, u16x2{0, 0}};
#pragma unroll
        for (int k = 0; k < KH; ++k) {
            if (page[k] < 0) gone |= 1 << k;
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int j = 0; j < (NB + 3) / 4; ++j) {
                    const uint32_t x = chk[k][e][j] & 0x7fff7fffu;
                    u16x2 y;
                    __builtin_memcpy(&y, &x, 4);
                    raw[e] = __builtin_elementwise_max(raw[e], y);
                }
        }
        const bool fails = max((int) raw[0][0], (int) raw[0][1]) >= (30 - sk) << 10 || max((int) raw[1][0], (int) raw[1][1]) >= (30 - sv) << 10;
        if (__any(fails)) {
            uint32_t top[2] = {0, 0};
#pragma unroll
            for (int k = 0; k < KH; ++k) {
                const int keys = page[k] < 0 ? 0 : len - 32 * (c + k);
                bool any_nan = false;
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int j = 0; j < NB / 2; ++j) {
                        uint32_t x = (chk[k][e][j / 2] >> (16 * (j & 1))) & 0x7fffu;
                        const int idx = l * (NB / 2) + j, key = 4 * (idx / (4 * NB)) + idx % 4;
                        x = key < keys ? x : 0u;
                        if (e) any_nan |= x > 0x7c00u;
                        top[e] = max(top[e], x > 0x7c00u ? 0u : x);
                    }
                if (__any(any_nan)) nans |= 1 << k;
            }
            sk = min(sk, 29 - (max_of_wave((int) top[0]) >> 10));   // exponent(d) + sk <= 14
            sv = min(sv, 29 - (max_of_wave((int) top[1]) >> 10));
        }
        const int mine = w / RN, keys = gone >> mine & 1 ? 0 : len - 32 * (c + mine);   // its cell, the request's keys in it
#pragma unroll
        for (int j = 0; j < PF; ++j) {
            const uint32_t d = mul_h2((uint32_t) kd[j] * 0x10001u, pow2_h2(sk)), c4 = kc[j], d4 = c4 >> 8;
            const uint32_t cc[4] = {codes<0>(c4), codes<1>(c4), codes<0>(d4), codes<1>(d4)};
            uint32_t hi[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) hi[e] = mul_h2(cc[e], d);
            *(u32x4*) operand(buf, mine, 0, kf + j) = u32x4{hi[0], hi[1], hi[2], hi[3]};
            if constexpr (EXACT)
                *(u32x4*) operand(buf, mine, 1, kf + j) =
                    u32x4{rest_h2(cc[0], d, hi[0]), rest_h2(cc[1], d, hi[1]), rest_h2(cc[2], d, hi[2]), rest_h2(cc[3], d, hi[3])};
        }
        uint32_t d[4];   // of keys (0, 2), (1, 3) of both halves
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            uint32_t x0 = vd[u][0], x1 = vd[u][1];
            if (keys < 32 || (nans >> mine & 1)) {   // keys behind the request's, NaNs: 0
                const int k0 = 16 * u + 4 * g;
                auto keep = [&](uint32_t x, int key) {
                    const uint32_t lo = (x & 0x7fffu) <= 0x7c00u && key < keys ? x & 0xffffu : 0u;
                    const uint32_t hi = (x >> 16 & 0x7fffu) <= 0x7c00u && key + 1 < keys ? x & 0xffff0000u : 0u;
                    return lo | hi;
                };
                x0 = keep(x0, k0);
                x1 = keep(x1, k0 + 2);
            }
            d[2 * u] = mul_h2(__builtin_amdgcn_perm(x1, x0, 0x05040100u), pow2_h2(sv));
            d[2 * u + 1] = mul_h2(__builtin_amdgcn_perm(x1, x0, 0x07060302u), pow2_h2(sv));
        }
        const uint32_t x0 = vc[0], x1 = vc[1], y0 = x0 >> 8, y1 = x1 >> 8;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            if (PF == 1 && half != (role & 1)) continue;
            const uint32_t cc[4] = {half ? codes<1>(x0) : codes<0>(x0), half ? codes<1>(y0) : codes<0>(y0),
                                    half ? codes<1>(x1) : codes<0>(x1), half ? codes<1>(y1) : codes<0>(y1)};
            uint32_t hi[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) hi[e] = mul_h2(cc[e], d[e]);
            const int f = 2 * NB + 2 * vb + half;
            *(u32x4*) operand(buf, mine, 0, f) = u32x4{hi[0], hi[1], hi[2], hi[3]};
            if constexpr (EXACT)
                *(u32x4*) operand(buf, mine, 1, f) = u32x4{rest_h2(cc[0], d[0], hi[0]), rest_h2(cc[1], d[1], hi[1]),
                                                           rest_h2(cc[2], d[2], hi[2]), rest_h2(cc[3], d[3], hi[3])};
        }
    };
    if (steps > 0) {
        check_pages();
        load(0);
    }

    // this lane's rows
    int lim[NC];
    h8 q[NC][NS][NB];
    float qs[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        const int r = r0 + n * RC + m;
        const bool ok = r < rows;
        lim[n] = ok ? back + (int) ((unsigned) r / R) : -1;
        qs[n] = 512.0f * qx[n].parts(a, ok, q[n]);
    }
    f4 o[NC][2 * NB];            // O^T 2^(osv - 9)
    float off[NC], mx[NC], lsum[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        off[n] = mx[n] = NO_KEY;
        lsum[n] = 0.0f;
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) o[n][i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    int osv = 15;
    auto ahead = [&](int step) __attribute__((always_inline)) {
        if (step + 1 < steps) {
            form(step + 1, (step & 1) ^ 1);
            if (step + 2 < steps) load(step + 2);
        }
    };
    auto multiply = [&](int buf, int c, int csk, int csv, bool nan_here) __attribute__((always_inline)) {
        const bool masked = 32 * c + 31 > every;                // some row does not see some key of the cell
        const int key0 = 32 * c + 4 * g;                        // key i of half u: key0 + 16 u + i
        f4 sc[NC][2];
#pragma unroll
        for (int n = 0; n < NC; ++n) sc[n][0] = sc[n][1] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        // Two operands a turn, the next turn's read ahead of this one's products; products that add to one
        // register stand 2 NC apart.
        constexpr int TURNS = NB * PARTS;
        auto read2 = [&](int f, int stride, int part, h8 (&x)[2]) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < 2; ++u) x[u] = *(const h8*) operand(buf, kh, part, f + u * stride);
        };
        h8 x[2][2];
        read2(0, NB, 0, x[0]);
#pragma unroll
        for (int i = 0; i < TURNS; ++i) {
            if (i + 1 < TURNS) read2((i + 1) / PARTS, NB, (i + 1) % PARTS, x[(i + 1) & 1]);
            else read2(2 * NB, 1, 0, x[(i + 1) & 1]);   // (the values' first)
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < NS; ++e)
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int n = 0; n < NC; ++n)
                        if (i % PARTS + e < 2)
                            sc[n][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[i & 1][u], q[n][e][i / PARTS], sc[n][u], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
        const float unit = bitsf((uint32_t) (127 - csk) << 23);
        if (csv != osv) {
            const float f = bitsf((uint32_t) (127 + csv - osv) << 23);
            osv = csv;
#pragma unroll
            for (int n = 0; n < NC; ++n)
#pragma unroll
                for (int i = 0; i < 2 * NB; ++i) o[n][i] *= f;
        }
        u32x4 pw[NC][NS];
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            const float qn = qs[n] * unit;
            if (masked)
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    sc[n][i / 4][i % 4] = key0 + 16 * (i / 4) + i % 4 <= lim[n] ? sc[n][i / 4][i % 4] : -INFINITY;
            float p[8], most = -INFINITY;
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = __builtin_fmaf(sc[n][i / 4][i % 4], qn, -off[n]);
#pragma unroll
            for (int i = 0; i < 8; ++i) most = fmaxf(most, p[i]);
            if (__any(most > 12.0f)) {
                float smax = sc[n][0][0];
#pragma unroll
                for (int i = 1; i < 8; ++i) smax = fmaxf(smax, sc[n][i / 4][i % 4]);
                mx[n] = fmaxf(mx[n], max_over_groups(smax) * qn);
                const float now = mx[n] == NO_KEY ? NO_KEY : mx[n] - 4.0f, f = exp2_hw(off[n] - now);
                off[n] = now;
                lsum[n] *= f;
#pragma unroll
                for (int i = 0; i < 2 * NB; ++i) o[n][i] *= f;
#pragma unroll
                for (int i = 0; i < 8; ++i) p[i] = __builtin_fmaf(sc[n][i / 4][i % 4], qn, -off[n]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                p[i] = exp2_hw(p[i]);
                lsum[n] += p[i];
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {   // keys i and i + 2 of each half
                const float p0 = p[4 * (k / 2) + k % 2], p1 = p[4 * (k / 2) + k % 2 + 2];
                const uint32_t hi = word_of((_Float16) p0, (_Float16) p1);
                pw[n][0][k] = hi;
                if (NS == 2) pw[n][NS - 1][k] = word_of((_Float16) less_half<0>(p0, hi), (_Float16) less_half<1>(p1, hi));
            }
        }
#pragma unroll
        for (int i = 0; i < TURNS; ++i) {
            const int at = TURNS + i;
            if (i + 1 < TURNS) read2(2 * NB + 2 * ((i + 1) / PARTS), 1, (i + 1) % PARTS, x[(at + 1) & 1]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < NS; ++e)
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int n = 0; n < NC; ++n)
                        if (i % PARTS + e < 2) {
                            f4& d = o[n][2 * (i / PARTS) + u];
                            d = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[at & 1][u], as_h8(pw[n][e][0], pw[n][e][1], pw[n][e][2], pw[n][e][3]), d, 0, 0, 0);
                        }
            __builtin_amdgcn_sched_barrier(0);
        }
        if (nan_here) {
            const uint8_t* cell = head + (int64_t) pages[c >> cpp] * page_bytes + (c & ((1 << cpp) - 1)) * (36 * D);
            for (int t = 0; t < 32; ++t)
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const uint16_t d = *(const uint16_t*) (cell + 34 * D + (((t >> 2) * NB + b) * 4 + (t & 3)) * 2);
                    if ((d & 0x7fffu) <= 0x7c00u) continue;
#pragma unroll
                    for (int n = 0; n < NC; ++n)
                        if (32 * c + t <= lim[n])
                            o[n][2 * b] = o[n][2 * b + 1] = f4{NAN, NAN, NAN, NAN};
                }
        }
    };
    if (steps > 0) form(0, 0);
    if (steps > 1) load(1);
    for (int step = 0; step < steps; ++step) {
        const int buf = step & 1, c = zc + step * KH + kh;
        const int csk = sk, csv = sv;
        const bool nan_here = nans >> kh & 1, work = !(gone >> kh & 1) && 32 * c <= last;   // some row of the wave sees the cell
        lds_barrier();   // this step's operands are there; the other buffer's readers are done
        // one of a SIMD's two waves forms operands while the other multiplies
        if (w < 4) ahead(step);
        if (work) {
            __builtin_amdgcn_s_setprio(1);
            multiply(buf, c, csk, csv, nan_here);
            __builtin_amdgcn_s_setprio(0);
        }
        if (w >= 4) ahead(step);
    }
    const float unit = bitsf((uint32_t) (127 + 9 - osv) << 23);
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        lsum[n] = sum_over_groups(lsum[n]);
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) {
            o[n][i] *= unit;
        }
    }
    if constexpr (KH == 2) {   // the second half's sums to the first
        lds_barrier();
        if (kh == 1) {
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                s_off[rg][n][l] = off[n];
                s_l[rg][n][l] = lsum[n];
#pragma unroll
                for (int i = 0; i < 2 * NB; ++i) *(f4*) (s_mem + (((rg * NC + n) * 2 * NB + i) * 64 + l) * 16) = o[n][i];
            }
        }
        lds_barrier();
        if (kh == 1) return;
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            const float other = s_off[rg][n][l], now = fmaxf(off[n], other), f0 = exp2_hw(off[n] - now), f1 = exp2_hw(other - now);
            off[n] = now;
            lsum[n] = lsum[n] * f0 + s_l[rg][n][l] * f1;
#pragma unroll
            for (int i = 0; i < 2 * NB; ++i)
                o[n][i] = o[n][i] * f0 + *(const f4*) (s_mem + (((rg * NC + n) * 2 * NB + i) * 64 + l) * 16) * f1;
        }
    }
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        const int r = r0 + n * RC + m;
        if (r >= rows) continue;
        const int tok = (int) ((unsigned) r / R), h = hd * (int) R + (int) ((unsigned) r % R), lastc = (back + tok) >> 5;
        if (lastc < a.row_cells) {   // the row's keys are all in the first split
            if (z > 0) continue;
            const float inv = lsum[n] == 0.0f ? 0.0f : 1.0f / lsum[n];
            char* dst = (char*) a.out + (int64_t) (s.row0 + tok) * a.out_nb1;
#pragma unroll
            for (int i = 0; i < 2 * NB; ++i) q4_put4(dst, a.type, h * D + 16 * i + 4 * g, o[n][i] * inv);
        } else if (zc <= lastc) {
            const int64_t p = ((int64_t) z * a.T + s.row0 + tok) * a.n_head + h;
#pragma unroll
            for (int i = 0; i < 2 * NB; ++i) *(f4*) (a.row_part + p * D + 16 * i + 4 * g) = o[n][i];
            if (g == 0) *(float2*) (a.row_stat + 2 * p) = float2{off[n], lsum[n]};
        }
    }
}

// Four dims of a row's sum so far: of the weights 2^(s - at) and of their products.
struct Q4Sum {
    f4 v = f4{0.0f, 0.0f, 0.0f, 0.0f};
    float at = NO_KEY, sum = 0.0f;
    __device__ __forceinline__ void add(const f4& pv, float pat, float psum) {
        const float now = fmaxf(at, pat), f0 = exp2_hw(at - now), f1 = exp2_hw(pat - now);
        v = v * f0 + pv * f1;
        sum = sum * f0 + psum * f1;
        at = now;
    }
    __device__ __forceinline__ void add(const float* part, const float* stat, int64_t p, int D, int dim) {
        const float2 st = *(const float2*) (stat + 2 * p);
        add(*(const f4*) (part + p * D + dim), st.x, st.y);
    }
    __device__ __forceinline__ f4 value() const { return v * (sum == 0.0f ? 0.0f : 1.0f / sum); }
};

// A row's splits, joined: a workgroup per row, D / 4 lanes per split; each lane adds every
// WAYS-th split in order, then the ways are added in order.
template <int D>
__device__ __forceinline__ void q4_join(const AttnQ4Args& a, int tok, int h, int parts, const float* part, const float* stat, int64_t row,
                                        int64_t heads) {
    constexpr int LN = D / 4, WAYS = 256 / LN;
    __shared__ __align__(16) f4 s_v[256];
    __shared__ float s_at[WAYS], s_sum[WAYS];
    const int tid = threadIdx.x, way = tid / LN, dim = 4 * (tid % LN);
    Q4Sum v;
#pragma unroll 4
    for (int z = way; z < parts; z += WAYS) v.add(part, stat, z * heads + row, D, dim);
    s_v[tid] = v.v;
    if (dim == 0) {
        s_at[way] = v.at;
        s_sum[way] = v.sum;
    }
    __syncthreads();
    if (way > 0) return;
    for (int k = 1; k < WAYS; ++k) v.add(s_v[k * LN + tid], s_at[k], s_sum[k]);
    q4_put4((char*) a.out + (int64_t) tok * a.out_nb1, a.type, h * D + dim, v.value());
}
__device__ __forceinline__ int q4_parts(int lim, int64_t cells) { return lim < 0 ? 1 : (int) ((unsigned) (lim >> 5) / (unsigned) cells) + 1; }

// of k_attn_q4: workgroups (request, head, token)
template <int D>
__global__ void __launch_bounds__(256) k_attn_q4_join(AttnQ4Args a, int most) {
    Q4Seq s;
    const int h = blockIdx.y, t = blockIdx.z;
    const int2 first = a.units ? a.first[blockIdx.x] : int2{(int) blockIdx.x, (int) a.cells};   // (not set: not used)
    if (!q4_request(a, blockIdx.x, s) || t >= s.n || !q4_fits(a, s) || (int64_t) s.n * (a.n_head / a.c.n_head_kv) > most) return;
    const int parts = q4_parts(s.len - s.n + t, first.y);
    if (parts > 1)
        q4_join<D>(a, s.row0 + t, h, parts, a.part, a.stat, ((int64_t) first.x * a.tcap + t) * a.n_head + h, (a.units ? 1 : a.S) * a.tcap * a.n_head);
}
// of k_attn_q4_rows: workgroups (token row, 1024 / D heads), D / 4 lanes a row: there are rows
// enough, so each lane adds its splits in order (two splits of 16384 rows of 128: 5.8 us; a
// workgroup per row as above 18.9).
template <int D>
__global__ void __launch_bounds__(256) k_attn_q4_rows_join(AttnQ4Args a, int most) {
    constexpr int LN = D / 4;
    Q4Seq s;
    const int tid = threadIdx.x, tok = blockIdx.x, h = blockIdx.y * (256 / LN) + tid / LN, dim = 4 * (tid % LN);
    if (!q4_find(a, tid & 63, tok, [](int t, int) { return (int64_t) t; }, s)) return;
    if (tok >= s.row0 + s.n || !q4_fits(a, s) || (int64_t) s.n * (a.n_head / a.c.n_head_kv) <= most) return;
    const int parts = q4_parts(s.len - s.n + (tok - s.row0), a.row_cells);
    if (parts == 1 || h >= a.n_head) return;
    const int64_t row = (int64_t) tok * a.n_head + h, rows = a.T * a.n_head;
    Q4Sum v;
#pragma unroll 2
    for (int z = 0; z < parts; ++z) v.add(a.row_part, a.row_stat, z * rows + row, D, dim);
    q4_put4((char*) a.out + (int64_t) tok * a.out_nb1, a.type, h * D + dim, v.value());
}

// Requests of up to `few` rows (eight tiles) are k_attn_q4's, the others k_attn_q4_rows', each kernel passing over the
// other's; one beyond max_new is k_attn_q4's where that runs.  A lone request that may have more rows is
// k_attn_q4_rows' whatever it has: one launch, not two.
template <int D, int NS>
int launch(const AttnQ4Args& a, hipStream_t st) {
    constexpr int W = q4_waves(D);
    const int few = a.tcap > 0 ? Q4_TILES * (16 / NS) : 0;
    const unsigned nk = (unsigned) a.c.n_head_kv;
    if (few) {
        hipLaunchKernelGGL((k_attn_q4<D, NS>), a.units ? dim3((unsigned) a.units, nk) : dim3((unsigned) a.S, nk, (unsigned) a.splits), dim3(64 * W), 0, st, a);
        if (a.splits > 1 || a.units)
            hipLaunchKernelGGL(k_attn_q4_join<D>, dim3((unsigned) a.S, (unsigned) a.n_head, (unsigned) a.tcap), dim3(256), 0, st, a, few);
    }
    if (few == 0 || std::min(a.max_new, a.T) * (a.n_head / a.c.n_head_kv) > few) {
        const int64_t blocks = q4_row_blocks(a);
        if (blocks > 0x7fffffff) return -2;
        const dim3 g((unsigned) blocks, nk, (unsigned) a.row_splits);
        if (a.type == KV_BF16) {
            if constexpr (NS == 1) hipLaunchKernelGGL((k_attn_q4_rows<D, 1, false>), g, dim3(512), 0, st, a, few);
        } else hipLaunchKernelGGL((k_attn_q4_rows<D, NS, true>), g, dim3(512), 0, st, a, few);
        if (a.row_splits > 1)
            hipLaunchKernelGGL(k_attn_q4_rows_join<D>, dim3((unsigned) a.T, (unsigned) ((a.n_head * (D / 4) + 255) / 256)), dim3(256), 0, st, a, few);
    }
    return hipGetLastError() == hipSuccess ? 0 : -3;
}
int parts_of(const AttnQ4Args& a) { return a.type == KV_F32 ? 8 : 16; }   // rows of a 16-column tile
int few_of(const AttnQ4Args& a) { return Q4_TILES * parts_of(a); }

}  // namespace

int64_t q4_few_tokens(const AttnQ4Args& a) {
    if (a.S == 1 && std::min(a.max_new, a.T) * (a.n_head / a.c.n_head_kv) > few_of(a)) return 0;
    return std::min<int64_t>(std::min(a.max_new, a.T), few_of(a) / (a.n_head / a.c.n_head_kv));
}
int64_t q4_splits(const AttnQ4Args& a) {
    if (q4_few_tokens(a) == 0) return 1;
    const int64_t groups = (int64_t) a.S * a.c.n_head_kv, cells = (a.max_len + KV_CELL - 1) / KV_CELL;
    const int64_t rows = q4_few_tokens(a) * (a.n_head / a.c.n_head_kv), W = q4_waves(a.c.D);
    int64_t tiles = 1;
    while (tiles < Q4_TILES && tiles * parts_of(a) < rows) tiles *= 2;
    // A workgroup to a CU (512: 131072 keys 29.2 us instead of 24.0), but twice as many for several requests of one tile, which
    // are seldom all as long as the longest (256: 24 ragged requests 26 us instead of 17.9); two cells to a wave at least.
    const int64_t want = a.S > 1 && tiles == 1 ? 512 : 256;
    return std::max<int64_t>(1, std::min<int64_t>(want / groups, cells / (2 * (W / tiles))));
}
// Requests of several lengths: their cells shared out on the device, to as many workgroups as fit the card once, or in
// whole rounds of it from half as many again as there are requests on (every request needs one).  us against
// uniform splits up to max_len: 24 requests of dozens to 8000 keys 11.5 and 17.9, 64 of them 26.6 and 46, 24 of 4000 all 21.0
// and 24.0, 60 of 2000 all 29 and 25.8.  Up to 64 requests, one to a lane: with four to a lane 200 ragged
// requests took 48 us, without splits 34, and 24 lost 0.5.
int q4_units(const AttnQ4Args& a, int& least) {
    if (q4_few_tokens(a) == 0 || a.S == 1 || a.S > 64) return 0;
    const int64_t cells = (a.max_len + KV_CELL - 1) / KV_CELL, rows = q4_few_tokens(a) * (a.n_head / a.c.n_head_kv);
    int tiles = 1;
    while (tiles < Q4_TILES && (int64_t) tiles * parts_of(a) < rows) tiles *= 2;
    least = q4_waves(a.c.D) / tiles;
    if (cells <= 2 * least || a.c.n_head_kv > 256) return 0;
    const int64_t round = 256 / a.c.n_head_kv;
    return (int) (round * ((3 * a.S + 2 * round - 1) / (2 * round)));
}
int64_t q4_row_blocks(const AttnQ4Args& a) {
    const int per = 8 / qr_halves(a.c.D) * qr_tiles(a.c.D) * 16;
    return a.T * (a.n_head / a.c.n_head_kv) / per + a.S;
}
int64_t q4_row_splits(const AttnQ4Args& a) {
    if (std::min(a.max_new, a.T) * (a.n_head / a.c.n_head_kv) <= few_of(a)) return 1;
    // As near to a workgroup per CU as whole splits come, of eight cells at least.  A 512-token f32 chunk in 2 splits (264
    // workgroups): 49.5 + 5.8 us, in 3 68.8 + 6.9, in 1 75; 100 tokens in 6 splits of 8 cells 27.7 + 4.7, in 3 of 16 35.8 + 4.6.
    const int64_t groups = q4_row_blocks(a) * a.c.n_head_kv, cells = (a.max_len + KV_CELL - 1) / KV_CELL;
    return std::max<int64_t>(1, std::min<int64_t>((256 + groups / 2) / groups, cells / 8));
}

int launch_attn_q4(const AttnQ4Args& a, hipStream_t st) {
    if (a.T == 0) return 0;
    const bool two = a.type == KV_F32;
    switch (a.c.D) {
        case 64: return two ? launch<64, 2>(a, st) : launch<64, 1>(a, st);
        case 128: return two ? launch<128, 2>(a, st) : launch<128, 1>(a, st);
        default: return two ? launch<256, 2>(a, st) : launch<256, 1>(a, st);
    }
}

}  // namespace qw
