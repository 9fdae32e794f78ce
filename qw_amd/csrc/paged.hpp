// paged.hpp - a pool of KV pages shared by many sequences, and what its kernels have in common.
//
// A page holds page_size tokens of every KV head; a table [n_seq][table_width] of page indices says
// where token t of a sequence lies: slot t % page_size of page table[b][t / page_size]. Indices
// outside the pool name no page: nothing is written there, and keys there take no part. Layouts are
// those the attention's matrix instructions take without a shuffle (E = 128 / bits codes in a
// 16-byte piece):
//   K  [page][head][slot][D * bits / 8 bytes]: the row's 32-dim steps c = d / 32, of each of which
//      lane group g = d % 32 / 8 takes 8 dims; piece i of group g at 64 i + 16 g, holding the 8 dims
//      of its 16 / bits steps one after another. fp16: dims in order. 8 bits: bytes in order. 4 bits: the
//      8 codes at nibbles v4_nibble_pos.
//   V  [page][head][slot / 8][D][8 codes]: for each dim the codes of 8 keys, 16, 8 or 4 bytes, in
//      the same order.
//   scales and biases of K and of V, [page][head][slot / 8][2][NG][8] fp16 (int8: the scales alone,
//      [1][1][8]), NG = D / 64.
// A 4- or 8-bit code in the low bits of a half is the subnormal code * 2^-24, which the matrix
// instructions take as it is: codes need a mask, no conversion, and the scales go to the scores and
// to the softmax weights.
// Beside them, for each page and head: the least and the largest key of every dim over what was
// written since slot 0 last was ([2][D] fp16), the same as 8-bit codes over the page's largest
// magnitude ([2][D], largest first), and that magnitude.
#pragma once

#include "kv_cache.hpp"

namespace qw {

struct PagedView {
    char* k;
    char* v;
    f16* k_par;
    f16* v_par;
    f16* lohi;
    int8_t* codes;
    float* top;
    int hkv, n_pages, lg;  // page_size = 1 << lg
};

struct PagedCache {
    int mode = QW_KV_FP16, bits = 16, D = 0, hkv = 0, n_pages = 0, page_size = 0, device = 0;
    PagedView view{};

    bool int8() const { return mode == QW_KV_INT8; }
    int par_halves() const { return bits == 16 ? 0 : int8() ? 8 : 2 * (D / kGroup) * 8; }  // of 8 slots
    int64_t nbytes() const;
    int init(int mode, int group_size, int n_kv_heads, int head_dim, int n_pages, int page_size, int device);
    void release();
};

// The sequences' places: table, the first position of each, the tokens of each.
struct PagedSeqs {
    const int32_t* table;
    int64_t stride;
    int width, n_seq;
    const int32_t* offsets;  // [n_seq + 1], or null: `each` tokens a sequence
    int each;
    const int32_t* starts;
    int n_tokens;

    // Runs of `size` slots that a sequence's tokens can touch, where each has as many of them.
    __host__ __device__ int runs(int size) const { return each == 1 ? 1 : (int)(((int64_t)each + size - 2) / size) + 1; }
};

int paged_update(PagedCache& c, const void* k, const void* v, int64_t k_token, int64_t k_head, int64_t v_token,
                 int64_t v_head, const PagedSeqs& s, hipStream_t stream);
int paged_gather(const PagedCache& c, void* k_out, void* v_out, const PagedSeqs& s, hipStream_t stream);
int check_seqs(const PagedCache& c, const PagedSeqs& s, const char* what);

// Queries [n_seq][n_q_heads][n_rows][D] of element strides, over the sequences' first lengths[b] keys.
struct PagedQuery {
    const void* q;
    int64_t seq_stride, head_stride, row_stride;
    int n_seq, n_q_heads, n_rows;
    const int32_t* lengths;
    const int32_t* table;
    int64_t table_stride;
    int table_width;
};
int check_query(const PagedCache& c, const PagedQuery& q, const char* what);
// picked (or null): [n_seq][hkv][n_picked] positions in the sequences' rows of the table.
int paged_attention(PagedCache& c, const PagedQuery& q, const int32_t* picked, int n_picked, float scale, void* out,
                    hipStream_t stream);

// The budget pages of each sequence and KV head that its queries' bounds rank first (paged_select.hip).
int paged_select(PagedCache& c, const PagedQuery& q, int budget, int sink, int recent, int32_t* picked, hipStream_t stream);

// Rotary positions of several axes (rope_axes.hip): positions [n_axes][n_tokens] (device), the axis of each pair (host).
struct RopeAxes {
    const int32_t* positions;
    int64_t stride;
    int n_axes;
    const uint8_t* axes;
    int rope_dims, traditional;
    float base, scale;
};
// What the kernels take of it, checked.
constexpr int kMaxHalf = 256;  // pairs
struct RopeTurns {
    const int32_t* positions;
    int64_t stride;  // of an axis
    int half, traditional;
    double log2_base, scale;  // scale over 2 pi
    uint8_t axes[kMaxHalf];
};
int rope_turns(const RopeAxes& r, int n_tokens, int hq, int hkv, int D, RopeTurns& out);
int rope_axes(const RopeAxes& r, const void* qkv, int n_tokens, int hq, int hkv, int D, void* q_out, void* k_out,
              hipStream_t stream);
// Tokens rotated on their way into their pages (paged_store.hip); half a multiple of 4.
int paged_turn_update(PagedCache& c, const RopeTurns& r, const void* qkv, int hq, void* q_out, const PagedSeqs& s,
                      hipStream_t stream);
int paged_rope_update(PagedCache& c, const RopeAxes& r, const void* qkv, int hq, void* q_out, const PagedSeqs& s,
                      hipStream_t stream);

// ------------------------------------------------------------------ device

// Turns a position of pair p, and the cosine and sine of one.
__device__ __forceinline__ double turn_rate(const RopeTurns& r, int p) {
    return exp2(-((double)p / r.half) * r.log2_base) * r.scale;
}
__device__ __forceinline__ float2 turn_of(double rate, int position) {
    double x = (double)position * rate;
    x -= rint(x);
    // what the angle's rounding to fp32 leaves turns them a little further: of 6.1M rotated values 915 differ from
    // the 64-bit result's rounding (without 1848; cosines in 64 bits 693, but 4 % slower)
    const float y = 2.0f * (float)x, rest = (float)(2.0 * x - (double)y) * 3.14159265f;
    float s, c;
    sincospif(y, &s, &c);
    return float2{__builtin_fmaf(-s, rest, c), __builtin_fmaf(c, rest, s)};
}

// Inclusive sums over a wave's lanes.
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
    // within rows of 16 lanes, then the rows' last lanes to the rows behind
    x += __builtin_amdgcn_update_dpp(0u, x, 0x111, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0u, x, 0x112, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0u, x, 0x114, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0u, x, 0x118, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0u, x, 0x142, 0xA, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0u, x, 0x143, 0xC, 0xF, false);
    return x;
}

// Which of n sequences holds unit `i` where sequence b has count(b) of them, and its index there; b = -1
// behind the last. Every lane of a wave calls it and gets the same.
struct PagedUnit {
    int b;
    uint32_t at, base;  // base: units before the sequence
};
// (from sequence b0 on, before which lie `base` units)
template <class F>
__device__ __forceinline__ PagedUnit find_unit(int n, uint32_t i, F count, int b0 = 0, uint32_t base = 0) {
    const int lane = (int)__lane_id();
    PagedUnit u{-1, 0u, 0u};
    auto in = [&](int at, uint32_t c) {  // (c: sequence at + lane's)
        const uint32_t s = wave_scan(c);
        const uint64_t past = __ballot(base + s > i);
        if (past) {
            const int l = __builtin_ctzll(past);
            u.base = base + (uint32_t)__builtin_amdgcn_readlane((int)(s - c), l);
            u.b = __builtin_amdgcn_readfirstlane(at + l);
            u.at = i - u.base;
        }
        base += (uint32_t)__builtin_amdgcn_readlane((int)s, 63);
        return past != 0;
    };
    constexpr int AHEAD = 4;  // of many, these times 64 at once
    for (; n - b0 > 64; b0 += 64 * AHEAD) {
        uint32_t c[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; k++) {
            const int b = b0 + 64 * k + lane;
            c[k] = count(min(b, n - 1));
            c[k] = b < n ? c[k] : 0u;
        }
#pragma unroll
        for (int k = 0; k < AHEAD; k++)
            if (in(b0 + 64 * k, c[k])) return u;
    }
    if (b0 < n) in(b0, b0 + lane < n ? count(b0 + lane) : 0u);
    return u;
}

// Where sequence b's new tokens go: positions start .. start + n - 1, from token `first` on.
struct PagedSpan {
    int start, n, first;
};
__device__ __forceinline__ PagedSpan span_of(const PagedSeqs& s, int b, int lg) {
    PagedSpan p;
    p.start = s.starts[b];
    int64_t lo, hi;
    if (s.offsets) {
        lo = s.offsets[b], hi = s.offsets[b + 1];
    } else {
        lo = (int64_t)b * s.each, hi = lo + s.each;
    }
    lo = lo < 0 ? 0 : lo;
    hi = hi > s.n_tokens ? s.n_tokens : hi;
    int64_t n = hi - lo;
    n = n < 0 || p.start < 0 ? 0 : n;
    p.n = (int)n;
    p.first = (int)(n > 0 ? lo : 0);
    return p;
}
// (the tokens behind the table's last page have no place)
__device__ __forceinline__ int span_in_table(const PagedSeqs& s, const PagedSpan& p, int lg) {
    const int64_t room = ((int64_t)s.width << lg) - p.start;
    return room < p.n ? (room > 0 ? (int)room : 0) : p.n;
}

}  // namespace qw
