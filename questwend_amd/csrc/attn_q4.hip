// attn_q4.hip -- causal attention of a batch of requests over the paged 4-bit cache
// (layout in qw_kv_q4.hpp): row (token t of n, query head h) of request i sees its keys
// 0 .. len - n + t,
//   o = sum_j softmax_j(scale q . k_j) v_j.
//
// Codes become f16 operands of v_mfma_f32_16x16x32_f16 in registers, without LDS: a code
// masked out of its dword is the f16 subnormal c 2^-24 (or, a nibble further on, c 2^-20), for
// two codes at once, and one packed multiply-add makes that (c - 8) 2^-9, exactly: nine
// instructions for eight operands.  (The subnormals themselves multiply too, but the
// products' sum then keeps 16 bits only.)  Block scales are applied in fp32 around
// the products, so the cache's values enter unrounded:
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
// A workgroup of four waves takes a block of a request's rows (R = n_head / n_head_kv rows
// per token) of one kv head and one split of the keys; each wave NC tiles of the rows, or,
// where the block has rows for one wave only, a quarter of the cells (their sums meet in
// LDS).  The next cell's dwords are loaded while this one's are computed on.
#include <algorithm>
#include <type_traits>

#include "../../include/qwmoe.h"
#include "qw_kv_q4.hpp"

namespace qw {

namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

constexpr float NO_KEY = -3.0e38f;   // M and off of a row that has seen no key yet

__device__ __forceinline__ void q4_put4(void* p, int type, int64_t i, f4 v) {
    if (type == KV_F32) *(f4*) ((float*) p + i) = v;
    else if (type == KV_F16) *(h4*) ((_Float16*) p + i) = __builtin_convertvector(v, h4);
    else *(b4*) ((__bf16*) p + i) = __builtin_convertvector(v, b4);
}

__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// The request that holds a block of rows (`per` rows a block, R rows per token): request
// i's blocks are numbered from floor(seq_start[i] R / per) + i on, which leaves room for
// every one of its blocks whatever the lengths, and is known without a prefix sum.
struct Q4Seq {
    int i, n, len;     // request, its new tokens, its keys (0: rows of zeros)
    int64_t row0;      // its first token row
};
__device__ __forceinline__ int64_t q4_block0(const AttnQ4Args& a, int i, int R, int per) {
    const int64_t t = min(max((int64_t) a.seq_start[i], (int64_t) 0), a.T);
    return t * R / per + i;
}
// The last of 0 .. n - 1 that `ok` holds for (it holds up to some place and not beyond), -1:
// none.  Called by whole waves, 64 candidates at a time.
template <typename F>
__device__ __forceinline__ int q4_last(int n, int lane, F ok) {
    int lo = 0, step = (n + 63) / 64;
    for (;;) {
        const int i = lo + lane * step;
        const uint64_t m = __ballot(i < n && ok(min(i, n - 1)));
        if (m == 0) return -1;
        lo = uni(lo + (__popcll(m) - 1) * step);
        if (step == 1) return lo;
        step = (step + 63) / 64;
    }
}
__device__ __forceinline__ bool q4_request(const AttnQ4Args& a, int i, Q4Seq& s) {
    if (i < 0) return false;
    const int64_t t0 = a.seq_start[i], t1 = a.seq_start[i + 1];
    s.i = i;
    s.row0 = t0;
    if (t0 < 0 || t1 > a.T || t1 <= t0) return false;
    s.n = (int) (t1 - t0);
    s.len = a.seq_len[i];
    return true;
}
// Whether the request's lengths fit the call.
__device__ __forceinline__ bool q4_fits(const AttnQ4Args& a, const Q4Seq& s) {
    return s.len >= 0 && s.len <= a.max_len && s.n <= a.max_new;
}

// One cell's dwords as they lie in memory.
template <int D>
struct Q4Cell {
    static constexpr int NB = D / 32;
    uint32_t k[2][NB];          // key codes of token l % 16 of both halves, dims 8 (l / 16) .. of each block
    uint32_t v[NB][2];          // value codes of dims l % 16 and 16 + l % 16 of each block, keys 4 (l / 16) ..
    uint32_t ks[2][NB][2];      // scales of keys 4 (l / 16) .. + 3 of both halves
    uint32_t vs[2][NB][2];
    uint32_t chk[(NB + 3) / 4]; // the lane's share of the value scales (NB / 2 halves)

    __device__ __forceinline__ void load(const uint8_t* cell, int l) {
        const int m = l & 15, g = l >> 4;
#pragma unroll
        for (int u = 0; u < 2; ++u) __builtin_memcpy(k[u], cell + (uint32_t) (((16 * u + m) * 4 + g) * NB * 4), 4 * NB);
#pragma unroll
        for (int u = 0; u < 2; ++u) __builtin_memcpy(ks[u], cell + (uint32_t) (16 * D + (4 * u + g) * NB * 8), 8 * NB);
#pragma unroll
        for (int b = 0; b < NB; b += 2)
            __builtin_memcpy(v[b], cell + (uint32_t) (18 * D + (((b / 2) * 16 + m) * 4 + g) * 16), 16);
#pragma unroll
        for (int u = 0; u < 2; ++u) __builtin_memcpy(vs[u], cell + (uint32_t) (34 * D + (4 * u + g) * NB * 8), 8 * NB);
        if constexpr (NB == 2) chk[0] = *(const uint16_t*) (cell + (uint32_t) (34 * D + 2 * l));
        else __builtin_memcpy(chk, cell + (uint32_t) (34 * D + NB * l), NB);
    }
    // the largest magnitude among the lane's halves of keys below `keys`, as f16 bits; NaNs count as 0
    __device__ __forceinline__ uint32_t top(int l, int keys, bool all) const {
        uint32_t t = 0;
#pragma unroll
        for (int e = 0; e < NB / 2; ++e) {
            uint32_t x = (chk[e / 2] >> (16 * (e & 1))) & 0x7fffu;
            const int at = l * (NB / 2) + e, key = 4 * (at / (4 * NB)) + at % 4;
            x = x > 0x7c00u || (!all && key >= keys) ? 0u : x;
            t = max(t, x);
        }
        return t;
    }
};

__device__ __forceinline__ float half_of(uint32_t w, int hi) {
    h2 x;
    __builtin_memcpy(&x, &w, 4);
    return (float) x[hi];
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

// (lane l ^ 8 of the same 16)
__device__ __forceinline__ float other_part(float v) { return dpp_f<0x128>(v); }   // row_ror:8

// NS f16 parts per row (f32 rows: two), NC tiles of 16 / NS rows per wave.
template <int D, int NS, int NC>
__global__ void __launch_bounds__(256) k_attn_q4(AttnQ4Args a) {
    constexpr int NB = D / 32, RC = 16 / NS, RW = NC * RC;
    constexpr int LD = D + 4;                                   // floats of a row in LDS
    __shared__ __align__(16) float s_o[4 * RC * LD];
    __shared__ float s_off[4][NC * RC], s_l[4][NC * RC];
    const int tid = threadIdx.x, l = tid & 63, m = l & 15, g = l >> 4;
    const int w = uni(tid >> 6);
    const int R = a.n_head / a.c.n_head_kv, hd = blockIdx.y, z = blockIdx.z;
    Q4Seq s;
    if (!q4_request(a, q4_last(a.S, l, [&](int i) { return q4_block0(a, i, R, 4 * RW) <= blockIdx.x; }), s)) return;
    const int64_t rows = (int64_t) s.n * R, base = ((int64_t) blockIdx.x - q4_block0(a, s.i, R, 4 * RW)) * (4 * RW);
    if (base >= rows) return;
    int len = s.len;
    if (!q4_fits(a, s)) {
        len = 0;
        if (tid == 0) atomicOr(a.status, QWMOE_STATUS_BAD_SEQ);
    }
    const bool share = rows - base <= RW;                       // rows for one wave only: its cells go to all four
    const int64_t r0 = base + (share ? 0 : w * RW);             // the wave's first row
    const int wrows = (int) max(min(rows - r0, (int64_t) RW), (int64_t) 0);
    const int wtiles = (wrows + RC - 1) / RC;
    const int back = len - s.n;                                 // a row of token t sees keys .. back + t
    const int last = wrows ? back + (int) ((r0 + wrows - 1) / R) : -1;   // the last key some row of the wave sees
    const int every = back + (int) (r0 / R);                    // keys up to here are seen by all of its rows
    const int cells = last < 0 ? 0 : (last >> 5) + 1;
    const int cshift = share ? 2 : 0;                           // the wave's cells: c0, c0 + 2^cshift ..
    const int c0 = (int) min((int64_t) z * a.cells + (share ? w : 0), (int64_t) cells);
    const int c1 = (int) min((int64_t) (z + 1) * a.cells, (int64_t) cells);
    const int block_last = back + (int) ((min(rows, base + 4 * RW) - 1) / R);
    if (z > 0 && (int64_t) z * a.cells > (block_last >> 5)) return;   // (z = 0 writes the rows without keys)

    // this lane's rows
    int lim[NC];            // the last key its row sees
    h8 q[NC][NB];
    float qs[NC];           // the scores' factor: scale log2(e), 2^9 for the codes, q's power of two
    int64_t orow[NC];       // token row * n_head + head, -1 without one
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        const bool ok = n * RC + (m % RC) < wrows;
        const int64_t r = ok ? r0 + n * RC + (m % RC) : 0;
        const int t = (int) (r / R), h = hd * R + (int) (r % R);
        orow[n] = ok ? (s.row0 + t) * a.n_head + h : -1;
        lim[n] = ok ? back + t : -1;
        float x[NB][8];
        const char* src = (const char*) a.q + (s.row0 + t) * a.q_nb1;
        const int64_t at = (int64_t) h * D + 8 * g;
        if constexpr (NS == 2) {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const f4 lo = *(const f4*) ((const float*) src + at + 32 * b), hi = *(const f4*) ((const float*) src + at + 32 * b + 4);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[b][j] = j < 4 ? lo[j & 3] : hi[j & 3];
            }
        } else {
            const bool f16 = a.type == KV_F16;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const u32x4 v = *(const u32x4*) ((const uint16_t*) src + at + 32 * b);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t word = v[j / 2];
                    x[b][j] = f16 ? half_of(word, j & 1) : bitsf(j & 1 ? word & 0xffff0000u : word << 16);
                }
            }
        }
        float big = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[b][j] = ok ? x[b][j] : 0.0f;
                big = fmaxf(big, __builtin_fabsf(x[b][j]));
            }
        big = fmaxf(big, __shfl_xor(big, 16));
        big = fmaxf(big, __shfl_xor(big, 32));
        // 2^ex <= big < 2^(ex + 1): q 2^(14 - ex) lies in f16's upper range
        const int ex = min(max((int) (fbits(big) >> 23) - 127, -100), 100);
        const float up = bitsf((uint32_t) (127 + 14 - ex) << 23);
        qs[n] = a.scale * bitsf((uint32_t) (127 - 5 + ex) << 23);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            h8 part;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float y = x[b][j] * up;
                _Float16 v = (_Float16) y;
                if (NS == 2 && m >= RC) v = (_Float16) (y - (float) v);
                part[j] = v;
            }
            q[n][b] = part;
        }
    }

    f4 o[NC][2 * NB];            // O^T 2^-9: dims 16 tile + 4 g + i of the lane's row
    float off[NC], mx[NC], lsum[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        off[n] = mx[n] = NO_KEY;
        lsum[n] = 0.0f;
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) o[n][i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    int E = -25;                 // the value scales so far are at most 2^E
    uint32_t Ebits = 0;          // 2^E as f16 bits

    const int32_t* pages = a.table + (int64_t) s.i * a.W;
    const int cpp = a.c.page_shift - 5;                         // log2 of a page's cells
    int pg = 0, pg_at = c0;                                     // the pages of 64 of the wave's cells, one per lane
    auto fetch_pages = [&](int c) {
        pg_at = c;
        const int mine = c + (l << cshift);
        pg = mine < c1 ? pages[mine >> cpp] : 0;
        if (pg < 0 || pg >= a.c.n_pages) {
            atomicOr(a.status, QWMOE_STATUS_BAD_SLOT);
            pg = -1;
        }
    };
    auto page_of = [&](int c) { return __builtin_amdgcn_readlane(pg, (c - pg_at) >> cshift); };
    auto address = [&](int c, int page) {
        return a.c.data + (int64_t) max(page, 0) * a.c.page_bytes() + hd * a.c.head_bytes() +
               (int64_t) (c & ((1 << cpp) - 1)) * (36 * D);
    };

    auto step = [&](const Q4Cell<D>& x, int c, bool gone, auto masked) __attribute__((always_inline)) {
        constexpr bool MASK = decltype(masked)::value;          // some row does not see some key of the cell
        f4 sc[NC][2];
#pragma unroll
        for (int n = 0; n < NC; ++n) sc[n][0] = sc[n][1] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const uint32_t c4 = x.k[u][b], d4 = c4 >> 8;
                const h8 ka = as_h8(codes<0>(c4), codes<1>(c4), codes<0>(d4), codes<1>(d4));
#pragma unroll
                for (int n = 0; n < NC; ++n) {
                    if (n && n >= wtiles) continue;   // uniform
                    const f4 p = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, q[n][b], f4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        sc[n][u][i] = __builtin_fmaf(p[i], half_of(x.ks[u][b][i / 2], i & 1), sc[n][u][i]);
                }
            }
        const uint32_t top = x.top(l, last + 1 - 32 * c, !MASK);
        bool move = top > Ebits;
        const float most = 12.0f - (float) E;
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            if (n && n >= wtiles) continue;
            float smax = -INFINITY;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float v = sc[n][u][i];
                    if (NS == 2) v += other_part(v);
                    if (MASK) v = !gone && 32 * c + 16 * u + 4 * g + i <= lim[n] ? v : -INFINITY;
                    sc[n][u][i] = v;
                    smax = fmaxf(smax, v);
                }
            move |= __builtin_fmaf(smax, qs[n], -off[n]) > most;
        }
        if (__any(move)) {
            uint32_t t = top;
#pragma unroll
            for (int k = 32; k >= 1; k >>= 1) t = max(t, (uint32_t) __shfl_xor((int) t, k));
            t = (uint32_t) uni((int) t);
            if (t > Ebits) {   // the power of two above the largest scale (from 2^-14 on, f16's smallest normal number)
                E = max((int) (t >> 10), 1) - 14;
                Ebits = (uint32_t) (E + 15) << 10;
            }
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                if (n && n >= wtiles) continue;
                float smax = -INFINITY;
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) smax = fmaxf(smax, sc[n][u][i]);
                smax = fmaxf(smax, __shfl_xor(smax, 16));
                smax = fmaxf(smax, __shfl_xor(smax, 32));
                mx[n] = fmaxf(mx[n], smax * qs[n]);
                const float now = mx[n] == NO_KEY ? NO_KEY : mx[n] + (float) (E - 4);
                const float f = exp2_hw(off[n] - now);
                off[n] = now;
                lsum[n] *= f;
#pragma unroll
                for (int i = 0; i < 2 * NB; ++i) o[n][i] *= f;
            }
        }
        // weights, formed in place
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            if (n && n >= wtiles) continue;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = exp2_hw(__builtin_fmaf(sc[n][u][i], qs[n], -off[n]));
                    sc[n][u][i] = p;
                    lsum[n] += p;
                }
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            h8 va[2];
            {
                const uint32_t x0 = x.v[b][0], x1 = x.v[b][1], y0 = x0 >> 8, y1 = x1 >> 8;
                va[0] = as_h8(codes<0>(x0), codes<0>(y0), codes<0>(x1), codes<0>(y1));
                va[1] = as_h8(codes<1>(x0), codes<1>(y0), codes<1>(x1), codes<1>(y1));
            }
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                if (n && n >= wtiles) continue;
                uint32_t pw[4];
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {   // keys i and i + 2
                        const float p0 = sc[n][u][i], p1 = sc[n][u][i + 2];
                        float d0 = half_of(x.vs[u][b][0], i), d1 = half_of(x.vs[u][b][1], i);
                        if (MASK) {   // (a masked key's scale may be a NaN)
                            const int key = 32 * c + 16 * u + 4 * g + i;
                            d0 = !gone && key <= lim[n] ? d0 : 0.0f;
                            d1 = !gone && key + 2 <= lim[n] ? d1 : 0.0f;
                        }
                        uint32_t hi = word_of((_Float16) (p0 * d0), (_Float16) (p1 * d1));
                        if (NS == 2) {
                            // (one rounding of the product for both uses: the compiler may round it in one step or in two)
                            asm volatile("" : "+v"(hi));
                            const uint32_t lo = word_of((_Float16) __builtin_fmaf(p0, d0, -half_of(hi, 0)),
                                                        (_Float16) __builtin_fmaf(p1, d1, -half_of(hi, 1)));
                            hi = m < RC ? hi : lo;
                        }
                        pw[2 * u + i] = hi;
                    }
                const h8 pb = as_h8(pw[0], pw[1], pw[2], pw[3]);
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    o[n][2 * b + k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va[k], pb, o[n][2 * b + k], 0, 0, 0);
            }
        }
    };
    {
        Q4Cell<D> x[2];
        int page[2] = {0, 0};
        int c = c0;
        if (c < c1) {
            fetch_pages(c);
            page[0] = page_of(c);
            x[0].load(address(c, page[0]), l);
        }
        auto turn = [&](int now) __attribute__((always_inline)) {
            const int next = c + (1 << cshift);
            if (next < c1) {
                if ((next - pg_at) >> cshift >= 64) fetch_pages(next);
                page[now ^ 1] = page_of(next);
                x[now ^ 1].load(address(next, page[now ^ 1]), l);
            }
            const bool gone = page[now] < 0;
            if (32 * c + 31 <= every && !gone) step(x[now], c, false, std::false_type{});
            else step(x[now], c, gone, std::true_type{});
            c = next;
        };
        while (c < c1) {
            turn(0);
            if (c >= c1) break;
            turn(1);
        }
    }

    // a row's results: out, or the split's sums
    const int64_t heads = a.T * a.n_head;
    auto put = [&](int64_t row, int lm, int dim, f4 v, float sum, float at) {
        const int parts = lm < 0 ? 1 : (int) ((lm >> 5) / a.cells) + 1;
        if (z >= parts) return;
        if (parts == 1) {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            char* dst = (char*) a.out + (row / a.n_head) * (int64_t) a.out_nb1;
            q4_put4(dst, a.type, (row % a.n_head) * D + dim, v * inv);
        } else {
            const int64_t p = z * heads + row;
            *(f4*) (a.part + p * D + dim) = v;
            if (dim == 0) *(float2*) (a.stat + 2 * p) = float2{at, sum};
        }
    };
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        lsum[n] += __shfl_xor(lsum[n], 16);
        lsum[n] += __shfl_xor(lsum[n], 32);
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) {
            o[n][i] *= 512.0f;
            if (NS == 2)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[n][i][j] += other_part(o[n][i][j]);
        }
    }
    if (!share) {
#pragma unroll
        for (int n = 0; n < NC; ++n)
            if (orow[n] >= 0 && m < RC)
#pragma unroll
                for (int i = 0; i < 2 * NB; ++i) put(orow[n], lim[n], 16 * i + 4 * g, o[n][i], lsum[n], off[n]);
        return;
    }
#pragma unroll
    for (int n = 0; n < NC; ++n)
        if (g == 0 && m < RC) {
            s_off[w][n * RC + m] = off[n];
            s_l[w][n * RC + m] = lsum[n];
        }
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        if (n * RC >= wrows) break;   // uniform over the workgroup
        __syncthreads();
        if (m < RC)
#pragma unroll
            for (int i = 0; i < 2 * NB; ++i) *(f4*) (s_o + (w * RC + m) * LD + 16 * i + 4 * g) = o[n][i];
        __syncthreads();
        for (int e = tid; e < RC * (D / 4); e += 256) {
            const int rr = e / (D / 4), dim = 4 * (e % (D / 4)), r = n * RC + rr;
            if (r >= wrows) break;
            const float at = fmaxf(fmaxf(s_off[0][r], s_off[1][r]), fmaxf(s_off[2][r], s_off[3][r]));
            f4 v = f4{0.0f, 0.0f, 0.0f, 0.0f};
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float f = exp2_hw(s_off[k][r] - at);
                v += *(const f4*) (s_o + (k * RC + rr) * LD + dim) * f;
                sum += s_l[k][r] * f;
            }
            const int64_t rq = r0 + r;
            const int t = (int) (rq / R);
            put((s.row0 + t) * a.n_head + hd * R + (int) (rq % R), back + t, dim, v, sum, at);
        }
    }
}

// A row's splits, joined: a workgroup per row, D / 4 lanes per split; each lane adds every
// WAYS-th split in order, then the ways are added in order.
template <int D>
__global__ void __launch_bounds__(256) k_attn_q4_join(AttnQ4Args a) {
    constexpr int LN = D / 4, WAYS = 256 / LN;
    __shared__ __align__(16) f4 s_v[256];
    __shared__ float s_at[WAYS], s_sum[WAYS];
    const int tid = threadIdx.x, way = tid / LN, dim = 4 * (tid % LN);
    const int64_t heads = a.T * a.n_head, row = blockIdx.x, tok = row / a.n_head;
    Q4Seq s;
    if (!q4_request(a, q4_last(a.S, tid & 63, [&](int i) { return a.seq_start[i] <= tok; }), s)) return;
    if (tok >= s.row0 + s.n || !q4_fits(a, s)) return;
    const int lim = s.len - s.n + (int) (tok - s.row0);
    const int parts = lim < 0 ? 1 : (int) ((lim >> 5) / a.cells) + 1;
    if (parts == 1) return;
    f4 v = f4{0.0f, 0.0f, 0.0f, 0.0f};
    float at = NO_KEY, sum = 0.0f;
    auto add = [&](const f4& pv, float pat, float psum) __attribute__((always_inline)) {
        const float now = fmaxf(at, pat), f0 = exp2_hw(at - now), f1 = exp2_hw(pat - now);
        v = v * f0 + pv * f1;
        sum = sum * f0 + psum * f1;
        at = now;
    };
#pragma unroll 4
    for (int z = way; z < parts; z += WAYS) {
        const int64_t p = z * heads + row;
        const float2 st = *(const float2*) (a.stat + 2 * p);
        add(*(const f4*) (a.part + p * D + dim), st.x, st.y);
    }
    s_v[tid] = v;
    if (dim == 0) {
        s_at[way] = at;
        s_sum[way] = sum;
    }
    __syncthreads();
    if (way > 0) return;
    for (int k = 1; k < WAYS; ++k) add(s_v[k * LN + tid], s_at[k], s_sum[k]);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    q4_put4((char*) a.out + tok * (int64_t) a.out_nb1, a.type, (row % a.n_head) * D + dim, v * inv);
}

template <int D, int NS, int NC>
int launch(const AttnQ4Args& a, hipStream_t st) {
    const int64_t blocks = q4_blocks(a, 4 * NC * (16 / NS));
    if (blocks > 0x7fffffff) return -2;
    const dim3 g((unsigned) blocks, (unsigned) a.c.n_head_kv, (unsigned) a.splits);
    hipLaunchKernelGGL((k_attn_q4<D, NS, NC>), g, dim3(256), 0, st, a);
    if (a.splits > 1) hipLaunchKernelGGL(k_attn_q4_join<D>, dim3((unsigned) (a.T * a.n_head)), dim3(256), 0, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -3;
}
template <int D, int NS>
int launch_tiles(const AttnQ4Args& a, hipStream_t st) {
    switch (q4_tiles(a)) {
        case 1: return launch<D, NS, 1>(a, st);
        case 2: return launch<D, NS, 2>(a, st);
        default:
            if constexpr (D < 256) return launch<D, NS, 4>(a, st);
            else return -2;
    }
}

}  // namespace

int q4_tiles(const AttnQ4Args& a) {
    const int64_t rows = std::min<int64_t>(a.max_new, a.T) * (a.n_head / a.c.n_head_kv), per = a.type == KV_F32 ? 8 : 16;
    return rows <= per ? 1 : rows <= 2 * per || a.c.D == 256 ? 2 : 4;
}
int64_t q4_blocks(const AttnQ4Args& a, int per) { return a.T * (a.n_head / a.c.n_head_kv) / per + a.S; }
int64_t q4_splits(const AttnQ4Args& a) {
    const int64_t per = (int64_t) 4 * q4_tiles(a) * (a.type == KV_F32 ? 8 : 16);
    const int64_t groups = q4_blocks(a, (int) per) * a.c.n_head_kv, cells = (a.max_len + KV_CELL - 1) / KV_CELL;
    return std::max<int64_t>(1, std::min<int64_t>({512 / groups, cells / 8, 4096}));
}

int launch_attn_q4(const AttnQ4Args& a, hipStream_t st) {
    if (a.T == 0) return 0;
    const bool two = a.type == KV_F32;
    switch (a.c.D) {
        case 64: return two ? launch_tiles<64, 2>(a, st) : launch_tiles<64, 1>(a, st);
        case 128: return two ? launch_tiles<128, 2>(a, st) : launch_tiles<128, 1>(a, st);
        default: return two ? launch_tiles<256, 2>(a, st) : launch_tiles<256, 1>(a, st);
    }
}

}  // namespace qw
