// qw_kv_q4.hpp -- the layout of the paged 4-bit key/value cache and the launches
// that read and write it.
//
// A page holds P = 2^page_shift tokens (P >= 32) as [kv head][P / 32 cells].  A cell
// is 32 tokens of one kv head: key codes (16 D bytes), key scales (2 D), value codes
// (16 D), value scales (2 D).  32 dimensions of a token's head are one block: a
// code 0 .. 15 per value and an f16 scale d, value = d (code - 8).  The order inside a
// cell is the one that the matrix-core attention loads without a shuffle: token
// 4 g + i (g, i = 0 .. 3) of 16-token tile u, block b of NB = D / 32,
//   key codes    dword ((16 u + 4 g + i) 4 + q) NB + b holds dims 32 b + 8 q + j, j = 0 .. 7,
//                at nibble j / 2 + 4 (j % 2): a pair of neighbouring dims is one mask away
//                from the two halves of a register;
//   value codes  dword ((((b / 2) 16 + j) 4 + g) 2 + b % 2) 2 + u, byte i: dim 32 b + j in the
//                low nibble, dim 32 b + 16 + j in the high one (a token's bytes are its own:
//                tokens are written without reading their neighbours);
//   scales       half ((4 u + g) NB + b) 4 + i.
#pragma once

#include "qw_common.hpp"

namespace qw {

constexpr int KV_CELL = 32;          // tokens of a cell
constexpr int KV_MAX_SEQ = 4096;     // requests of a call (the plan's lengths lie in LDS)
constexpr int KV_MAX_PAGE = 4096;    // tokens of a page

enum KvType : int { KV_F32 = 0, KV_F16 = 1, KV_BF16 = 30 };

struct KvQ4 {
    uint8_t* data;
    int n_head_kv, D, page_shift;
    int64_t n_pages;
    __host__ __device__ int64_t head_bytes() const { return ((int64_t) 36 * D) << (page_shift - 5); }
    __host__ __device__ int64_t page_bytes() const { return head_bytes() * n_head_kv; }
    // the cell of a slot (page * P + token in page), for head 0
    __device__ int64_t cell(int64_t slot) const {
        const int64_t page = slot >> page_shift;
        const int in = (int) (slot & ((1 << page_shift) - 1));
        return page * page_bytes() + (int64_t) (in >> 5) * (36 * D);
    }
};

template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ uint32_t kv_dpp(uint32_t v) {
    return (uint32_t) __builtin_amdgcn_update_dpp(0, (int) v, CTRL, ROWS, 0xF, true);
}
// Sums that stay at 2^32 - 1 once there: above every bound they are compared with (rows, pages
// and widths are below 2^31, as is each addend, so a sum that matters is not clipped).
__device__ __forceinline__ uint32_t kv_add(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }
__device__ __forceinline__ uint32_t kv_wave_incl(uint32_t v) {   // sums over the lanes up to this one
    v = kv_add(v, kv_dpp<0x111>(v));
    v = kv_add(v, kv_dpp<0x112>(v));
    v = kv_add(v, kv_dpp<0x114>(v));
    v = kv_add(v, kv_dpp<0x118>(v));
    v = kv_add(v, kv_dpp<0x142, 0xA>(v));   // the last of row 0 to row 1, of row 2 to row 3
    return kv_add(v, kv_dpp<0x143, 0xC>(v));   // the last of row 1 to rows 2 and 3
}

struct KvPlanArgs {
    const int32_t *held, *past, *n_new;   // [S]
    int S, page_shift;
    int64_t n_pages;
    int32_t* table;                       // [S][W]
    int64_t W;
    int32_t* ring;                        // [n_pages]
    const int64_t* counters;              // head, tail
    int64_t* counters_out;
    int64_t T;
    int32_t *seq_start, *seq_len;         // [S + 1], [S]
    int64_t* slot;                        // [T]
    int32_t* pos;                         // [T]
    int32_t* status;
};
int launch_kv_plan(const KvPlanArgs& a, hipStream_t stream);

struct KvRowsArgs {
    KvQ4 c;
    int type;                             // KvType of the rows
    const void *k, *v;                    // rows of n_head_kv * D values, nb1 bytes apart (store)
    void *ko, *vo;                        // (load)
    size_t k_nb1, v_nb1;
    const int64_t* slot;                  // [T]; negative: the row is passed over
    int64_t T;
    int32_t* status;
};
int launch_kv_q4_store(const KvRowsArgs& a, hipStream_t stream);
int launch_kv_q4_load(const KvRowsArgs& a, hipStream_t stream);

struct AttnQ4Args {
    KvQ4 c;
    int type;
    const void* q;                        // [T][n_head][D], tokens q_nb1 bytes apart
    void* out;                            // likewise
    size_t q_nb1, out_nb1;
    int n_head, S;
    int group;                            // query heads per kv head, and 2^32 / group rounded up
    uint32_t group_inv;
    int64_t T, W;
    const int32_t *table, *seq_start, *seq_len;
    int64_t max_new, max_len;
    float scale;                          // of the scores, times log2(e)
    // requests of few rows: cells of 32 keys per split, and where there is more than one, their
    // sums [splits][S][tcap][n_head][D] and [..][2] offset and sum of weights
    int64_t cells, tcap;
    int splits;
    // or, units > 0: splits by the lengths at hand, `least` cells or more each, `units` of them or fewer for
    // all requests together; their sums are [units][tcap][n_head][..], a request's first one and cells per split
    // first[i]
    int units, least;
    int2* first;
    float *part, *stat;
    // the others: likewise, [row_splits][T][n_head][..]
    int64_t row_cells;
    int row_splits;
    float *row_part, *row_stat;
    int32_t* status;
};
int64_t q4_few_tokens(const AttnQ4Args& a);   // new tokens, at most, of a request of few rows
int64_t q4_splits(const AttnQ4Args& a);       // splits of the keys that fill the card
int q4_units(const AttnQ4Args& a, int& least);   // (as in AttnQ4Args)
int64_t q4_row_splits(const AttnQ4Args& a);
int64_t q4_row_blocks(const AttnQ4Args& a);
int launch_attn_q4(const AttnQ4Args& a, hipStream_t stream);

}  // namespace qw
