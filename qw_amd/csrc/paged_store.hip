// paged_store.hip - new tokens into their pages, quantized, and back out as fp16.
//
// The codecs are the caches' own: MLX affine in groups of 64 dims (quant.hpp), per-token int8, fp16.
// A workgroup takes one page of one head, so that every word that holds several keys' codes, and the
// page's bounds, have one writer. A wave takes 8 slots (two times 8 at D = 128): a lane holds 4 dims of
// 8 tokens of K and V, 16 lanes a group, whose extremes come by DPP. Those 16 lanes then each form the
// step and base of one of the 16 rows (8 tokens' K and V), with its divisions, and hand them round; codes come
// by a product and one correction of its remainder, and are packed as bytes as they are converted (two
// keys' 4-bit codes as one number), so that V's words of 8 keys need no transposition. Where a call
// covers part of such a word the rest is kept; tokens that a call does not have cost nothing. Bound by HBM where there are many
// (65536 int8 tokens, 8 heads of D = 128, pages of 32: 83 us, 5.1 TB/s, and read back 71, 5.7), by the chain of loads and some
// 1,100 instructions a wave where they fill the card once (6001 8-bit tokens, 4 heads of D = 256: 13.8 us, 2.8 TB/s). A token's
// heads lie on one XCD, 8 pages side by side.
#include <algorithm>

#include "paged.hpp"
#include "quant.hpp"
#include "rope.hpp"

namespace qw {

namespace {

size_t align16(size_t x) { return (x + 255) / 256 * 256; }

}  // namespace

int64_t PagedCache::nbytes() const {
    const int64_t ph = (int64_t)n_pages * hkv, rows = ph * page_size;
    return 2 * rows * D * bits / 8 + 2 * rows / 8 * par_halves() * 2 + ph * (4 * D + 2 * D + 4);
}

int PagedCache::init(int mode_, int group_size, int n_kv_heads, int head_dim, int n_pages_, int page_size_, int device_) {
    QW_REQUIRE(mode_ == QW_KV_FP16 || mode_ == QW_KV_AFFINE8 || mode_ == QW_KV_AFFINE4 || mode_ == QW_KV_INT8 ||
                   mode_ == QW_KV_TURBO4,
               QW_ERR_INVALID_ARGUMENT, "qw_paged_create: unknown mode");
    QW_REQUIRE(mode_ != QW_KV_TURBO4, QW_ERR_UNSUPPORTED, "qw_paged_create: turbo4 has no paged form");
    QW_REQUIRE(n_kv_heads > 0 && n_kv_heads <= 65535 && n_pages_ > 0, QW_ERR_INVALID_ARGUMENT,
               "qw_paged_create: 1 .. 65535 KV heads and at least one page expected");
    QW_REQUIRE(head_dim == 128 || head_dim == 256, QW_ERR_UNSUPPORTED, "qw_paged_create: head_dim 128 or 256");
    QW_REQUIRE((mode_ != QW_KV_AFFINE8 && mode_ != QW_KV_AFFINE4) || group_size == kGroup, QW_ERR_UNSUPPORTED,
               "qw_paged_create: affine modes use group_size 64");
    QW_REQUIRE(page_size_ >= 16 && page_size_ <= 256 && (page_size_ & (page_size_ - 1)) == 0, QW_ERR_UNSUPPORTED,
               "qw_paged_create: page_size 16, 32, 64, 128 or 256");
    mode = mode_;
    bits = mode == QW_KV_AFFINE4 ? 4 : mode == QW_KV_FP16 ? 16 : 8;
    D = head_dim;
    hkv = n_kv_heads;
    n_pages = n_pages_;
    page_size = page_size_;
    device = device_;
    DeviceGuard dg(device);
    QW_REQUIRE(dg.ok, QW_ERR_HIP, "qw_paged_create: hipSetDevice failed");
    const size_t ph = (size_t)n_pages * hkv, rows = ph * page_size;
    const size_t sizes[7] = {rows * D * bits / 8, rows * D * bits / 8, rows / 8 * par_halves() * 2, rows / 8 * par_halves() * 2,
                             ph * 4 * D, ph * 2 * D, ph * 4};
    void* at[7] = {};
    for (int i = 0; i < 7; i++) {
        const bool ok = sizes[i] == 0 || hipMalloc(&at[i], align16(sizes[i])) == hipSuccess;
        if (!ok) {
            (void)hipGetLastError();
            for (void* p : at)
                if (p) (void)hipFree(p);
            set_error("qw_paged_create: hipMalloc of " + std::to_string(sizes[i]) + " bytes failed");
            return QW_ERR_OUT_OF_MEMORY;
        }
    }
    view = PagedView{(char*)at[0], (char*)at[1], (f16*)at[2], (f16*)at[3], (f16*)at[4], (int8_t*)at[5], (float*)at[6],
                     hkv, n_pages, __builtin_ctz(page_size)};
    for (int i = 0; i < 7; i++)
        if (at[i]) QW_HIP_CHECK(hipMemset(at[i], 0, sizes[i]));
    QW_HIP_CHECK(hipDeviceSynchronize());
    return QW_OK;
}

void PagedCache::release() {
    if (!view.k) return;  // (a refused pool: no device call)
    DeviceGuard dg(device);
    (void)hipDeviceSynchronize();
    void* ptrs[7] = {view.k, view.v, view.k_par, view.v_par, view.lohi, view.codes, view.top};
    for (void* p : ptrs)
        if (p) (void)hipFree(p);
    view = PagedView{};
}

int check_seqs(const PagedCache& c, const PagedSeqs& s, const char* what) {
    const std::string w(what);
    QW_REQUIRE(s.n_tokens >= 0 && s.n_seq >= 0 && (s.n_tokens == 0 || s.n_seq > 0), QW_ERR_INVALID_ARGUMENT,
               w + ": n_tokens and n_seq >= 0, and a sequence for the tokens, expected");
    QW_REQUIRE(s.n_tokens == 0 || (s.table && s.starts && s.width > 0), QW_ERR_INVALID_ARGUMENT, w + ": null table/starts, or a table without columns");
    QW_REQUIRE(s.stride >= s.width, QW_ERR_INVALID_ARGUMENT, w + ": a table stride below its width");
    QW_REQUIRE((int64_t)s.width * c.page_size <= 0x7fffff00, QW_ERR_INVALID_ARGUMENT, w + ": table_width * page_size < 2^31 expected");
    QW_REQUIRE(s.n_seq <= 65535 && s.n_tokens <= (1 << 28), QW_ERR_UNSUPPORTED, w + ": at most 65535 sequences and 2^28 tokens a call");
    QW_REQUIRE(s.n_tokens == 0 || s.offsets || s.n_tokens % s.n_seq == 0, QW_ERR_INVALID_ARGUMENT,
               w + ": without offsets n_tokens is a multiple of n_seq");
    return QW_OK;
}

namespace {

// The greatest of a row: D / 4 lanes.
template <int D>
__device__ __forceinline__ float row_max(float x) {
    const int lane = (int)__lane_id();
    x = fmaxf(x, dpp_mov<0xB1>(x));
    x = fmaxf(x, dpp_mov<0x4E>(x));
    x = fmaxf(x, dpp_mov<0x124>(x));
    x = fmaxf(x, dpp_mov<0x128>(x));
    x = fmaxf(x, lane_xor<16>(x, lane));
    return D == 256 ? fmaxf(x, lane_xor<32>(x, lane)) : x;
}

// f of 0 .. 7, as constants.
template <class F>
__device__ __forceinline__ void each8(F f) {
    using std::integral_constant;
    f(integral_constant<int, 0>()), f(integral_constant<int, 1>()), f(integral_constant<int, 2>()), f(integral_constant<int, 3>());
    f(integral_constant<int, 4>()), f(integral_constant<int, 5>()), f(integral_constant<int, 6>()), f(integral_constant<int, 7>());
}

// Lane J's value to all 16 lanes of its row.
template <int J>
__device__ __forceinline__ float of_lane(float x) {
    return dpp_mov<0x150 + J>(x);
}

// Rows' extremes as pairs of halves, both of which the least is taken of (exact: the rows are halves): an affine row's least
// and negative greatest, or the negative magnitudes of a K and a V row.
// As written: the compiler puts an instruction before it for each operand, against signalling NaNs.
__device__ __forceinline__ half2v least(half2v a, half2v b) {
    half2v y;
    asm("v_pk_min_f16 %0, %1, %2" : "=v"(y) : "v"(a), "v"(b));
    return y;
}
__device__ __forceinline__ half2v least_negated(half2v a, half2v b) {  // of -a and -b
    half2v y;
    asm("v_pk_min_f16 %0, %1, %2 neg_lo:[1,1] neg_hi:[1,1]" : "=v"(y) : "v"(a), "v"(b));
    return y;
}
__device__ __forceinline__ half2v least_of_negative(half2v a, half2v b) {  // of a and -b
    half2v y;
    asm("v_pk_min_f16 %0, %1, %2 neg_lo:[0,1] neg_hi:[0,1]" : "=v"(y) : "v"(a), "v"(b));
    return y;
}
__device__ __forceinline__ half2v ends_of(half4v x) {
    const half2v a = least(x.lo, x.hi), b = least_negated(x.lo, x.hi);
    return least(half2v{a[0], b[0]}, half2v{a[1], b[1]});
}
__device__ __forceinline__ half2v sizes_of(half4v k, half4v v) {
    auto negative = [](half2v x) { return __builtin_bit_cast(half2v, __builtin_bit_cast(uint32_t, x) | 0x80008000u); };
    const half2v a = least(negative(k.lo), negative(k.hi)), b = least(negative(v.lo), negative(v.hi));
    return least(half2v{a[0], b[0]}, half2v{a[1], b[1]});
}
template <int CTRL>
__device__ __forceinline__ half2v moved(half2v x) {
    asm volatile("s_nop 1" : "+v"(x));  // (two waits between a write of x, which may be in assembly, and a lane move of it)
    return __builtin_bit_cast(half2v, dpp_mov<CTRL>(__builtin_bit_cast(float, x)));
}
template <int S>
__device__ __forceinline__ half2v lane_least(half2v x, int lane) {
    asm volatile("s_nop 1" : "+v"(x));
    return least(x, __builtin_bit_cast(half2v, lane_xor<S>(__builtin_bit_cast(float, x), lane)));
}
// The first N of x over as many lanes of 16: lane i ends with x[i]'s least. Each step leaves a lane half of its rows, and
// gives the other half to a lane that differs in the next bit (by mirrors for bits 3 and 2).
template <int N>
__device__ __forceinline__ half2v spread_least(half2v* x, int r16) {
    auto step = [&](auto half, auto ctrl) {
        constexpr int H = decltype(half)::value;
        const bool up = (r16 & H) != 0;
#pragma unroll
        for (int j = 0; j < H; j++) {
            const half2v keep = up ? x[j + H] : x[j], give = up ? x[j] : x[j + H];
            x[j] = least(keep, moved<decltype(ctrl)::value>(give));
        }
    };
    using std::integral_constant;
    if constexpr (N == 16) step(integral_constant<int, 8>(), integral_constant<int, 0x140>());
    step(integral_constant<int, 4>(), integral_constant<int, 0x141>());
    step(integral_constant<int, 2>(), integral_constant<int, 0x4E>());
    step(integral_constant<int, 1>(), integral_constant<int, 0xB1>());
    return x[0];
}

// Steps of the rows' codes: value = code * step + base, inv = 1 / step.
struct Steps {
    float step, base, inv;
};
template <int BITS, bool INT8>
__device__ __forceinline__ Steps steps_of(float mn, float mx, f16& scale, f16& bias) {
    if constexpr (INT8) {  // mx: the row's largest magnitude
        scale = (f16)(mx / 127.0f);
        if ((float)scale == 0.0f) scale = (f16)1.0f;
        bias = (f16)0.0f;
        return Steps{(float)scale, 0.0f, 1.0f / (float)scale};
    } else {
        const AffineGroup q = affine_group(mn, mx, BITS);
        scale = (f16)q.scale;
        bias = (f16)q.bias;
        return Steps{q.scale, q.bias, 1.0f / q.scale};
    }
}
// A code in a float: of 4 bits a whole number, of 8 bits before its rounding (put_byte rounds to the
// nearest, to even, and ends at 0 and 255). The quotient: inv is the step's reciprocal, rounded
// once; the product of it and its remainder, which an fma has exactly, correct it to the rounded quotient
// (Markstein, 1990), as the codec's division gives it. x finite. one: 1.0 that the compiler doesn't know, for a
// difference that takes x as a half.
template <int BITS>
__device__ __forceinline__ float code_of(f16 x, const Steps& q, float one) {
    const float t = __builtin_fmaf((float)x, one, -q.base);
    float p = t * q.inv;
    p = __builtin_fmaf(__builtin_fmaf(-p, q.step, t), q.inv, p);
    return BITS == 8 ? p : __builtin_amdgcn_fmed3f(__builtin_rintf(p), 0.0f, 15.0f);
}
// int8's, 128 above themselves, in the low bytes of two halves: the codec rounds the quotient to a half, and a half in
// 1024 .. 2047 ends at its ones, so that the sum with 1152 rounds it to the nearest, to even.
__device__ __forceinline__ uint32_t codes_of(half2v x, const Steps& q) {
    half2v y;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const float p = __builtin_fmaf((float)x[i], q.inv, 0.0f);
        y[i] = (f16)__builtin_fmaf(__builtin_fmaf(-p, q.step, (float)x[i]), q.inv, p);
    }
    y = __builtin_elementwise_min(__builtin_elementwise_max(y, half2v{} - (f16)128.0f), half2v{} + (f16)127.0f);
    return __builtin_bit_cast(uint32_t, y + (f16)1152.0f);
}
template <int BYTE>
__device__ __forceinline__ uint32_t put_byte(uint32_t w, float c) {
    return __builtin_amdgcn_cvt_pk_u8_f32(c, BYTE, w);
}

// Byte 64 i + 16 g + .. of a K row where a lane's 4 dims (of index li) begin.
template <int BITS>
__device__ __forceinline__ int k_at(int li) {
    const int c = li >> 3, g = (li & 7) >> 1, hi = li & 1;
    if (BITS == 16) return 8 * li;
    if (BITS == 8) return (c >> 1) * 64 + g * 16 + (c & 1) * 8 + hi * 4;
    return (c >> 2) * 64 + g * 16 + (c & 3) * 4;
}

// Run `i` of `size` slots: counted over the sequences' own runs where they have offsets, else over as many for each (of
// 1024 tokens of as many sequences 23.3 us when counted, 17 so).
template <class F>
__device__ __forceinline__ PagedUnit unit_of(const PagedSeqs& s, uint32_t i, int size, F count) {
    if (s.offsets) return find_unit(s.n_seq, i, count);
    const uint32_t per = s.runs(size), b = i / per;
    PagedUnit u{-1, i - b * per, 0u};
    if (b < (uint32_t)s.n_seq && u.at < count((int)b)) u.b = (int)b;
    return u;
}

constexpr int kStoreWaves = 8;

struct StoreArgs {
    const f16* k;
    const f16* v;
    int64_t k_token, k_head, v_token, v_head;
    PagedSeqs s;
};

// Rotates 4 dims d .. of heads.
struct Turner {
    double rate[4];
    float cos[4], sin[4];
    int d, p, other;  // its first pair, the dims of the pairs' other halves (itself: adjacent ones)
    bool turns, first, adjacent;

    __device__ __forceinline__ Turner(const RopeTurns& r, int d_) : d(d_), other(d_) {
        turns = d < 2 * r.half, first = d < r.half, adjacent = r.traditional != 0;
        if (!adjacent && turns) other = first ? d + r.half : d - r.half;
        p = adjacent ? d >> 1 : min(d, other);
        if (!turns) return;
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (e < (adjacent ? 2 : 4)) rate[e] = turn_rate(r, p + e);
    }
    __device__ __forceinline__ void at(const RopeTurns& r, int64_t token) {
        if (!turns) return;
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (e < (adjacent ? 2 : 4)) {
                const float2 t = turn_of(rate[e], r.positions[r.axes[p + e] * r.stride + token]);
                cos[e] = t.x, sin[e] = t.y;
            }
    }
    __device__ __forceinline__ half4v of(half4v x, half4v z) const {  // z: the other halves (not of adjacent pairs)
        if (!turns) return x;
        if (adjacent) z = half4v{x[1], x[0], x[3], x[2]};
        half4v y;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const bool one = adjacent ? e % 2 == 0 : first;
            const float c0 = cos[e / 2], c1 = cos[e], s0 = sin[e / 2], s1 = sin[e];
            float r1, r2;
            rope_rot((float)(one ? x[e] : z[e]), (float)(one ? z[e] : x[e]), adjacent ? c0 : c1, adjacent ? s0 : s1, r1, r2);
            y[e] = (f16)(one ? r1 : r2);
        }
        return y;
    }
};
struct TurnArgs {
    RopeTurns r;
    f16* q_out;
    int hq, groups;  // workgroups that store; those behind them rotate q, kTurnHeads heads of a token each
};
constexpr int kTurnHeads = 8;

// TURN: k rotates on its way, q in workgroups of its own.
template <int BITS, bool INT8, int D, bool TURN>
__global__ __launch_bounds__(64 * kStoreWaves) void paged_update_kernel(PagedView c, StoreArgs a, TurnArgs turn) {
    if constexpr (TURN) {
        if ((int)blockIdx.x >= turn.groups) {
            const int per = (turn.hq + kTurnHeads - 1) / kTurnHeads, i = (int)blockIdx.x - turn.groups;
            const int64_t token = i / per;
            const int h0 = i % per * kTurnHeads;
            Turner t(turn.r, threadIdx.x % (D / 4) * 4);
            t.at(turn.r, token);
            const f16* q = a.k - (int64_t)turn.hq * D + token * a.k_token;
            for (int h = h0 + threadIdx.x / (D / 4); h < min(h0 + kTurnHeads, turn.hq); h += blockDim.x / (D / 4))
                *(half4v*)(turn.q_out + (token * turn.hq + h) * D + t.d) = t.of(*(const half4v*)(q + h * D + t.d), *(const half4v*)(q + h * D + t.other));
            return;
        }
    }
    constexpr int LPR = D / 4, SUB = 64 / LPR, NG = INT8 ? 1 : D / kGroup;
    __shared__ half4v sm_lo[kStoreWaves][LPR], sm_hi[kStoreWaves][LPR];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    // (heads side by side on an XCD: a token's row of all heads is read at about the same time)
    const int nw = blockDim.x >> 6, h = (int)((blockIdx.x >> 3) % c.hkv), ps = 1 << c.lg;
    const PagedUnit u = unit_of(a.s, (blockIdx.x >> 3) / c.hkv * 8 + (blockIdx.x & 7), ps, [&](int b) {
        const PagedSpan p = span_of(a.s, b, c.lg);
        const int n = span_in_table(a.s, p, c.lg);
        return n > 0 ? (uint32_t)(((p.start + n - 1) >> c.lg) - (p.start >> c.lg) + 1) : 0u;
    });
    if (u.b < 0) return;
    const PagedSpan p = span_of(a.s, u.b, c.lg);
    const int n = span_in_table(a.s, p, c.lg);
    const int logical = (p.start >> c.lg) + (int)u.at;
    const int page = a.s.table[u.b * a.s.stride + logical];
    const int pos0 = logical << c.lg;
    const int s0 = max(p.start - pos0, 0), s1 = min(p.start + n - pos0, ps);
    const int64_t ph = (int64_t)page * c.hkv + h;
    const int li = lane % LPR, sub = lane / LPR, grp = li >> 4;

    const int r16 = lane & 15;
    const f16 inf = (f16)INFINITY;
    half4v lo = {inf, inf, inf, inf}, negative_hi = lo;
    const int first = s0 >> 3, last = (s1 - 1) >> 3;
    for (int b0 = first; b0 <= last; b0 += nw * SUB) {
        const int blk = b0 + wave * SUB + sub;
        half4v xk[8], xv[8];
        auto in = [&](int k) { return 8 * blk + k >= s0 && 8 * blk + k < s1; };
        const bool whole = 8 * blk >= s0 && 8 * blk + 8 <= s1;
        const int64_t t0 = (int64_t)p.first + (pos0 + 8 * blk - p.start);  // slot 8 blk's token, if that is the call's
        const f16* kt = a.k + t0 * a.k_token + h * a.k_head + 4 * li;
        const f16* vt = a.v + t0 * a.v_token + h * a.v_head + 4 * li;
        if (__all(whole)) {
#pragma unroll
            for (int k = 0; k < 8; k++) xk[k] = *(const half4v*)(kt + k * a.k_token), xv[k] = *(const half4v*)(vt + k * a.v_token);
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++) {
                xk[k] = half4v{}, xv[k] = half4v{};
                if (in(k)) xk[k] = *(const half4v*)(kt + k * a.k_token), xv[k] = *(const half4v*)(vt + k * a.v_token);
            }
        }
        if constexpr (TURN) {
            Turner t(turn.r, 4 * li);
            half4v z[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                z[k] = half4v{};
                if (in(k)) z[k] = *(const half4v*)(kt + k * a.k_token + (t.other - t.d));
            }
            each8([&](auto k) {
                constexpr int K = decltype(k)::value;
                if (!__any(in(K))) return;
                t.at(turn.r, in(K) ? t0 + K : p.first);
                xk[K] = t.of(xk[K], z[K]);
            });
        }
        if (page < 0 || page >= c.n_pages) return;  // (the whole workgroup's; the tokens were requested beside the table's entry)
        const bool live = blk <= last;
        const int64_t blk8 = ph * (ps >> 3) + blk;
        char* krow = c.k + (ph * ps + 8 * blk) * (D * BITS / 8) + k_at<BITS>(li);
        u32x4* vblk = (u32x4*)(c.v + blk8 * (D * BITS) + 4 * li * BITS);  // this lane's 4 dims
        // what the words hold of keys that this call leaves alone
        u32x4 old[BITS / 4];
#pragma unroll
        for (int j = 0; j < BITS / 4; j++) old[j] = live && !whole ? vblk[j] : u32x4{0, 0, 0, 0};
        auto bounds = [&](half4v x, bool with) {
            const half2v l0 = least(lo.lo, x.lo), l1 = least(lo.hi, x.hi);
            const half2v h0 = least_of_negative(negative_hi.lo, x.lo), h1 = least_of_negative(negative_hi.hi, x.hi);
            lo.lo = with ? l0 : lo.lo, lo.hi = with ? l1 : lo.hi;
            negative_hi.lo = with ? h0 : negative_hi.lo, negative_hi.hi = with ? h1 : negative_hi.hi;
        };
        if (__all(whole)) {
#pragma unroll
            for (int k = 0; k < 8; k++) bounds(xk[k], true);
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++) bounds(xk[k], in(k));
        }
        float cv[8][4];      // V's codes
        uint32_t cv2[8][2];  // int8's, of dims 0 1 and 2 3
        float one = 1.0f;
        asm volatile("" : "+v"(one));
        if constexpr (BITS == 16) {
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (in(k)) *(half4v*)(krow + k * (D * 2)) = xk[k];
        } else {
            // the rows' extremes: K's of token k in lane k of a group, V's in lane 8 + k
            float mn = 0.0f, mx;
            if constexpr (INT8) {
                half2v x[8];
#pragma unroll
                for (int k = 0; k < 8; k++) x[k] = sizes_of(xk[k], xv[k]);
                half2v y = spread_least<8>(x, r16);
                y = least(y, moved<0x128>(y));
                y = lane_least<16>(y, lane);
                if (D == 256) y = lane_least<32>(y, lane);
                mx = -(float)(r16 < 8 ? y[0] : y[1]);
            } else {
                half2v x[16];
#pragma unroll
                for (int k = 0; k < 8; k++) x[k] = ends_of(xk[k]), x[8 + k] = ends_of(xv[k]);
                const half2v y = spread_least<16>(x, r16);
                mn = (float)y[0], mx = -(float)y[1];
            }
            f16 scale, bias;
            const Steps mine = steps_of<BITS, INT8>(mn, mx, scale, bias);
            each8([&](auto k) {
                constexpr int K = decltype(k)::value;
                if (!__any(in(K))) {
#pragma unroll
                    for (int i = 0; i < 4; i++) cv[K][i] = 0.0f;
                    cv2[K][0] = cv2[K][1] = 0;
                    return;
                }
                const Steps qk{of_lane<K>(mine.step), of_lane<K>(mine.base), of_lane<K>(mine.inv)};
                const Steps qv{of_lane<8 + K>(mine.step), of_lane<8 + K>(mine.base), of_lane<8 + K>(mine.inv)};
                float c[4];
                if constexpr (INT8) {
                    cv2[K][0] = codes_of(xv[K].lo, qv), cv2[K][1] = codes_of(xv[K].hi, qv);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        c[i] = code_of<BITS>(xk[K][i], qk, one);
                        cv[K][i] = code_of<BITS>(xv[K][i], qv, one);
                    }
                }
                if constexpr (INT8) {
                    const uint32_t w = __builtin_amdgcn_perm(codes_of(xk[K].hi, qk), codes_of(xk[K].lo, qk), 0x06040200u);
                    if (in(K)) *(uint32_t*)(krow + K * D) = w;
                } else if constexpr (BITS == 4) {
                    // dims 8 j .. + 3 in an even lane (nibbles 0, 4, 1, 5), .. + 7 in the odd one (2, 6, 3, 7)
                    uint32_t w = put_byte<0>(0u, __builtin_fmaf(16.0f, c[2], c[0]));
                    w = put_byte<2>(w, __builtin_fmaf(16.0f, c[3], c[1]));
                    w |= __builtin_amdgcn_update_dpp(0u, w, 0xB1, 0xF, 0xF, false) << 8;  // the other lane's
                    if (in(K) && (li & 1) == 0) *(uint32_t*)(krow + K * (D / 2)) = w;
                } else {
                    const uint32_t w = put_byte<3>(put_byte<2>(put_byte<1>(put_byte<0>(0u, c[0]), c[1]), c[2]), c[3]);
                    if (in(K)) *(uint32_t*)(krow + K * D) = w;
                }
            });
            if (in(r16 & 7) && (!INT8 || li < 16)) {
                f16* par = (r16 < 8 ? c.k_par : c.v_par) + blk8 * (INT8 ? 8 : 16 * NG) + (INT8 ? 0 : 8 * grp) + (r16 & 7);
                par[0] = scale;
                if (!INT8) par[8 * NG] = bias;
            }
        }
        if (live) {
            uint32_t key[4];  // of key pair j: all bits of the halves that this call writes
#pragma unroll
            for (int j = 0; j < 4; j++) key[j] = (in(2 * j) ? 0xFFFFu : 0u) | (in(2 * j + 1) ? 0xFFFF0000u : 0u);
            if constexpr (BITS == 16) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    u32x4 w;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const uint32_t x = __builtin_bit_cast(uint32_t, half2v{xv[2 * j][i], xv[2 * j + 1][i]});
                        w[j] = (x & key[j]) | (old[i][j] & ~key[j]);
                    }
                    vblk[i] = w;
                }
            } else if constexpr (BITS == 8) {
                uint32_t m[2];
#pragma unroll
                for (int j = 0; j < 2; j++)
                    m[j] = (key[2 * j] & 0xFFu) | (key[2 * j] >> 8 & 0xFF00u) | (key[2 * j + 1] << 16 & 0xFF0000u) |
                           (key[2 * j + 1] & 0xFF000000u);
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        uint32_t x;
                        if constexpr (INT8) {
                            const uint32_t a = __builtin_amdgcn_perm(cv2[4 * j + 1][i / 2], cv2[4 * j][i / 2], 0x06020400u);
                            const uint32_t b = __builtin_amdgcn_perm(cv2[4 * j + 3][i / 2], cv2[4 * j + 2][i / 2], 0x06020400u);
                            x = __builtin_amdgcn_perm(b, a, i & 1 ? 0x07060302u : 0x05040100u);
                        } else {
                            x = put_byte<0>(0u, cv[4 * j][i]);
                            x = put_byte<1>(x, cv[4 * j + 1][i]);
                            x = put_byte<2>(x, cv[4 * j + 2][i]);
                            x = put_byte<3>(x, cv[4 * j + 3][i]);
                        }
                        const uint32_t o = old[i / 2][2 * (i & 1) + j];
                        old[i / 2][2 * (i & 1) + j] = (x & m[j]) | (o & ~m[j]);
                    }
                vblk[0] = old[0];
                vblk[1] = old[1];
            } else {
                uint32_t m = 0;
#pragma unroll
                for (int j = 0; j < 4; j++) m |= (key[j] & 0x000F000Fu) << (4 * j);
                u32x4 w;
#pragma unroll
                for (int i = 0; i < 4; i++) {  // nibbles of keys 0 2 | 4 6 | 1 3 | 5 7
                    uint32_t x = put_byte<0>(0u, __builtin_fmaf(16.0f, cv[2][i], cv[0][i]));
                    x = put_byte<1>(x, __builtin_fmaf(16.0f, cv[6][i], cv[4][i]));
                    x = put_byte<2>(x, __builtin_fmaf(16.0f, cv[3][i], cv[1][i]));
                    x = put_byte<3>(x, __builtin_fmaf(16.0f, cv[7][i], cv[5][i]));
                    w[i] = (x & m) | (old[0][i] & ~m);
                }
                vblk[0] = w;
            }
        }
    }
    // the page's bounds
    f16* lohi = c.lohi + ph * 2 * D + 4 * li;
    half4v hi = -negative_hi, was_lo = lo, was_hi = hi;
    if (s0 > 0 && wave == 0) was_lo = *(const half4v*)lohi, was_hi = *(const half4v*)(lohi + D);
    auto other_half = [&](half4v x) {
        const u32x2 u = __builtin_bit_cast(u32x2, x);
        return __builtin_bit_cast(half4v, u32x2{__float_as_uint(lane_xor<32>(__uint_as_float(u[0]), lane)),
                                                __float_as_uint(lane_xor<32>(__uint_as_float(u[1]), lane))});
    };
    if constexpr (SUB == 2) {
        lo = __builtin_elementwise_min(lo, other_half(lo));
        hi = __builtin_elementwise_max(hi, other_half(hi));
    }
    if (nw > 1) {
        if (sub == 0) sm_lo[wave][li] = lo, sm_hi[wave][li] = hi;
        __syncthreads();
        if (wave) return;
        for (int w = 1; w < nw; w++) {
            lo = __builtin_elementwise_min(lo, sm_lo[w][li]);
            hi = __builtin_elementwise_max(hi, sm_hi[w][li]);
        }
    }
    if (s0 > 0) {
        lo = __builtin_elementwise_min(lo, was_lo);
        hi = __builtin_elementwise_max(hi, was_hi);
    }
    const f16 most = (f16)65504.0f;
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        lo[i] = lo[i] < -most ? -most : lo[i] > most ? most : lo[i];
        hi[i] = hi[i] < -most ? -most : hi[i] > most ? most : hi[i];
        if (!(lo[i] <= hi[i])) lo[i] = hi[i] = (f16)0.0f;  // nothing but NaN
        top = fmaxf(top, fmaxf(fabsf((float)lo[i]), fabsf((float)hi[i])));
    }
    top = row_max<D>(top);
    const float inv = top > 0.0f ? 127.0f / top : 0.0f;
    uint32_t wl = 0, wh = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        wh |= ((uint32_t)(int)__builtin_amdgcn_fmed3f(__builtin_ceilf((float)hi[i] * inv), -127.0f, 127.0f) & 0xFFu) << (8 * i);
        wl |= ((uint32_t)(int)__builtin_amdgcn_fmed3f(__builtin_floorf((float)lo[i] * inv), -127.0f, 127.0f) & 0xFFu) << (8 * i);
    }
    if (sub == 0) {
        *(half4v*)lohi = lo;
        *(half4v*)(lohi + D) = hi;
        *(uint32_t*)(c.codes + ph * 2 * D + 4 * li) = wh;
        *(uint32_t*)(c.codes + ph * 2 * D + D + 4 * li) = wl;
    }
    if (lane == 0) c.top[ph] = top;
}

// 4 dims' fp16 values of a code word (a byte each): f16(f16(code * scale) + bias).
template <bool INT8>
__device__ __forceinline__ half4v values4(uint32_t w, f16 s, f16 b) {
    half4v y;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float c = (float)(int)(w >> (8 * i) & 0xFFu);
        y[i] = INT8 ? (f16)((c - 128.0f) * (float)s) : (f16)affine_dequant(c, s, b);
    }
    return y;
}

template <int BITS, bool INT8, int D>
__global__ __launch_bounds__(256) void paged_gather_kernel(PagedView c, PagedSeqs s, f16* k_out, f16* v_out) {
    constexpr int LPR = D / 4, SUB = 64 / LPR, NG = INT8 ? 1 : D / kGroup;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int h = (int)((blockIdx.x >> 3) % c.hkv), ps = 1 << c.lg;
    const int li = lane % LPR, sub = lane / LPR, grp = INT8 ? 0 : li >> 4;
    const uint32_t unit = (((blockIdx.x >> 3) / c.hkv * 8 + (blockIdx.x & 7)) * 4 + wave) * SUB;
    auto blocks = [&](int b) {
        const PagedSpan p = span_of(s, b, c.lg);
        return p.n > 0 ? (uint32_t)((((int64_t)p.start + p.n - 1) >> 3) - (p.start >> 3) + 1) : 0u;
    };
    PagedUnit u = unit_of(s, unit, 8, blocks);
    if (SUB == 1 && u.b < 0) return;
    if constexpr (SUB == 2) {
        const PagedUnit u1 = unit_of(s, unit + 1, 8, blocks);
        if (sub) u = u1;
        if (u.b < 0) return;
    }
    const PagedSpan p = span_of(s, u.b, c.lg);
    const int64_t pos0 = ((int64_t)(p.start >> 3) + u.at) * 8, end = (int64_t)p.start + p.n;
    const int64_t logical = pos0 >> c.lg;
    int page = logical < s.width ? s.table[u.b * s.stride + logical] : -1;
    const bool there = page >= 0 && page < c.n_pages;
    page = there ? page : 0;
    const int slot0 = (int)(pos0 & (ps - 1));
    const int64_t ph = (int64_t)page * c.hkv + h, blk8 = ph * (ps >> 3) + (slot0 >> 3);
    const char* krow = c.k + (ph * ps + slot0) * (D * BITS / 8) + k_at<BITS>(li);
    const u32x4* vblk = (const u32x4*)(c.v + blk8 * (D * BITS) + 4 * li * BITS);
    u32x4 vw[BITS / 4];
#pragma unroll
    for (int j = 0; j < BITS / 4; j++) vw[j] = vblk[j];
    half8 ks{}, kb{}, vs{}, vb{};
    if constexpr (BITS != 16) {
        const f16* kp = c.k_par + blk8 * (INT8 ? 8 : 16 * NG) + 8 * grp;
        const f16* vp = c.v_par + blk8 * (INT8 ? 8 : 16 * NG) + 8 * grp;
        ks = *(const half8*)kp, vs = *(const half8*)vp;
        if (!INT8) kb = *(const half8*)(kp + 8 * NG), vb = *(const half8*)(vp + 8 * NG);
    }
    half4v yk[8];
    uint32_t kw[8];
#pragma unroll
    for (int k = 0; k < 8; k++) {
        if constexpr (BITS == 16)
            yk[k] = *(const half4v*)(krow + k * (D * 2));
        else
            kw[k] = *(const uint32_t*)(krow + k * (D * BITS / 8));
    }
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const int64_t pos = pos0 + k;
        half4v y;
        if constexpr (BITS == 16) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t w = vw[i][k / 2];
                y[i] = __builtin_bit_cast(f16, (uint16_t)(k & 1 ? w >> 16 : w));
            }
        } else {
            uint32_t w = kw[k], x = 0;
            if constexpr (BITS == 4) {
                w >>= 8 * (li & 1);
                w = (w & 15u) | (w >> 16 & 15u) << 8 | (w >> 4 & 15u) << 16 | (w >> 20 & 15u) << 24;
#pragma unroll
                for (int i = 0; i < 4; i++) x |= (vw[0][i] >> (4 * v4_nibble_pos(k)) & 15u) << (8 * i);
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) x |= (vw[i / 2][2 * (i & 1) + k / 4] >> (8 * (k & 3)) & 0xFFu) << (8 * i);
            }
            yk[k] = values4<INT8>(w, ks[k], kb[k]);
            y = values4<INT8>(x, vs[k], vb[k]);
        }
        if (pos >= p.start && pos < end) {
            const int64_t at = ((int64_t)(p.first + (pos - p.start)) * c.hkv + h) * D + 4 * li;
            // (past the caches: 65536 int8 tokens with the store 168 us, so 151; the store's own rows and codes so 157)
            __builtin_nontemporal_store(there ? yk[k] : half4v{}, (half4v*)(k_out + at));
            __builtin_nontemporal_store(there ? y : half4v{}, (half4v*)(v_out + at));
        }
    }
}

template <class F>
void by_mode(const PagedCache& c, F f) {
    auto of = [&](auto bits, auto i8) {
        if (c.D == 256)
            f(bits, i8, std::integral_constant<int, 256>());
        else
            f(bits, i8, std::integral_constant<int, 128>());
    };
    using std::integral_constant;
    if (c.bits == 16)
        of(integral_constant<int, 16>(), integral_constant<bool, false>());
    else if (c.bits == 4)
        of(integral_constant<int, 4>(), integral_constant<bool, false>());
    else if (c.int8())
        of(integral_constant<int, 8>(), integral_constant<bool, true>());
    else
        of(integral_constant<int, 8>(), integral_constant<bool, false>());
}

// Runs of `size` slots that the tokens can touch.
int64_t most_units(const PagedSeqs& s, int size) {
    if (!s.offsets) return (int64_t)s.n_seq * s.runs(size);
    return std::min<int64_t>(s.n_tokens, (int64_t)s.n_tokens / size + 2 * (int64_t)s.n_seq);
}

int store_waves(const PagedCache& c, const PagedSeqs& s) {
    // waves for the blocks of 8 slots that an average sequence touches in a page, two a wave at D = 128. So many / 8 / 2 at
    // most, the store alone, replayed over the same tokens, us: a token each of 33 sequences, pages of 16, D = 128 4.6 / 7.5 / 4.6; 2048
    // each of 8, pages of 256 19.7 / 19.6 / 32.1; 13107 each of 5, pages of 32, Int8 63 / 163 / 64 (82 where they are in no cache)
    const int blocks = std::min(c.page_size / 8, s.n_tokens / s.n_seq / 8 + 1);
    return std::max(1, std::min(kStoreWaves, blocks * c.D / 256));
}

}  // namespace

int paged_update(PagedCache& c, const void* k, const void* v, int64_t k_token, int64_t k_head, int64_t v_token,
                 int64_t v_head, const PagedSeqs& s, hipStream_t stream) {
    if (int rc = check_seqs(c, s, "paged update")) return rc;
    if (s.n_tokens == 0) return QW_OK;
    QW_REQUIRE(k && v, QW_ERR_INVALID_ARGUMENT, "paged update: null k/v");
    QW_REQUIRE(((uintptr_t)k | (uintptr_t)v) % 8 == 0 && (k_token | k_head | v_token | v_head) % 4 == 0 && k_token >= 0 &&
                   k_head >= 0 && v_token >= 0 && v_head >= 0,
               QW_ERR_INVALID_ARGUMENT, "paged update: k and v 8-byte aligned with strides of whole 8 bytes expected");
    DeviceGuard dg(c.device);
    QW_REQUIRE(dg.ok, QW_ERR_HIP, "paged update: hipSetDevice failed");
    const StoreArgs a{(const f16*)k, (const f16*)v, k_token, k_head, v_token, v_head, s};
    const int waves = store_waves(c, s);
    const int64_t groups = (most_units(s, c.page_size) + 7) / 8 * 8 * c.hkv;
    QW_REQUIRE(groups * 64 * waves <= UINT32_MAX, QW_ERR_UNSUPPORTED, "paged update: too many tokens for one call");
    const dim3 grid((unsigned)groups);
    by_mode(c, [&](auto bits, auto i8, auto d) {
        hipLaunchKernelGGL((paged_update_kernel<decltype(bits)::value, decltype(i8)::value, decltype(d)::value, false>), grid,
                           dim3(64 * waves), 0, stream, c.view, a, TurnArgs{});
    });
    QW_HIP_CHECK(hipGetLastError());
    return QW_OK;
}

int paged_turn_update(PagedCache& c, const RopeTurns& r, const void* qkv, int hq, void* q_out, const PagedSeqs& s,
                      hipStream_t stream) {
    QW_REQUIRE(qkv && q_out && r.positions, QW_ERR_INVALID_ARGUMENT, "paged rope update: null qkv/positions/q_out");
    const int64_t row = (int64_t)(hq + 2 * c.hkv) * c.D;
    const f16* k = (const f16*)qkv + (int64_t)hq * c.D;
    const StoreArgs a{k, k + (int64_t)c.hkv * c.D, row, c.D, row, c.D, s};
    const int64_t groups = (most_units(s, c.page_size) + 7) / 8 * 8 * c.hkv;
    const int64_t all = groups + (int64_t)s.n_tokens * ((hq + kTurnHeads - 1) / kTurnHeads);
    const int waves = store_waves(c, s);
    QW_REQUIRE(all * 64 * waves <= UINT32_MAX, QW_ERR_UNSUPPORTED, "paged rope update: too many tokens for one call");
    const TurnArgs turn{r, (f16*)q_out, hq, (int)groups};
    by_mode(c, [&](auto bits, auto i8, auto d) {
        hipLaunchKernelGGL((paged_update_kernel<decltype(bits)::value, decltype(i8)::value, decltype(d)::value, true>),
                           dim3((unsigned)all), dim3(64 * waves), 0, stream, c.view, a, turn);
    });
    QW_HIP_CHECK(hipGetLastError());
    return QW_OK;
}

int paged_gather(const PagedCache& c, void* k_out, void* v_out, const PagedSeqs& s, hipStream_t stream) {
    if (int rc = check_seqs(c, s, "paged gather")) return rc;
    if (s.n_tokens == 0) return QW_OK;
    QW_REQUIRE(k_out && v_out, QW_ERR_INVALID_ARGUMENT, "paged gather: null k_out/v_out");
    QW_REQUIRE(((uintptr_t)k_out | (uintptr_t)v_out) % 8 == 0, QW_ERR_INVALID_ARGUMENT, "paged gather: outputs 8-byte aligned expected");
    DeviceGuard dg(c.device);
    QW_REQUIRE(dg.ok, QW_ERR_HIP, "paged gather: hipSetDevice failed");
    const int64_t per = 4 * 256 / c.D;  // units a workgroup
    const int64_t groups = (most_units(s, 8) + 8 * per - 1) / (8 * per) * 8 * c.hkv;
    QW_REQUIRE(groups * 256 <= UINT32_MAX, QW_ERR_UNSUPPORTED, "paged gather: too many tokens for one call");
    const dim3 grid((unsigned)groups);
    by_mode(c, [&](auto bits, auto i8, auto d) {
        hipLaunchKernelGGL((paged_gather_kernel<decltype(bits)::value, decltype(i8)::value, decltype(d)::value>), grid,
                           dim3(256), 0, stream, c.view, s, (f16*)k_out, (f16*)v_out);
    });
    QW_HIP_CHECK(hipGetLastError());
    return QW_OK;
}

}  // namespace qw
