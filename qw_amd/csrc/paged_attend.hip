// paged_attend.hip - attention of the newest tokens of many sequences over their pages.
//
// out = softmax(scale q . k) v for each row over its sequence's keys, causal among the last n_rows of
// them, in one pass with the running maximum and sum. Bound by reading the codes once from HBM.
//
// Work is dealt in rounds of 128 keys: the rounds of all sequences, one behind the other, in equal runs
// to the workers of a head (a grid sized for the card, lengths read on the device), so that sequences of
// any lengths keep the chip busy. A worker's piece of a sequence that is not all of it goes to a
// workspace as fp32 partials that a second launch joins.
//
// A wave takes 32 keys of a round, straight from memory into the matrix instructions' operands:
//   S^T = K Q^T: two tiles of 16 keys; tile t's row i is key 8 (i / 4) + 4 t + i % 4, so that lane
//     group g ends with the scores of keys 8 g .. 8 g + 7 of the query row that it holds, which is
//   O^T = V^T P^T's second operand as it stands; V's 8 codes of a dim are the first.
// Codes enter as subnormal halves (paged.hpp). A group's score is scale * (q . code) + bias * sum q; P
// is multiplied by a key's V scale in fp32 and rounded once to fp16; the biases' part is one more matrix
// product, of P with the biases.
// The next round's K is requested behind this one's scores, its V behind this one's P V: a wave
// always waits for loads that are half a round old.
#include <algorithm>

#include "paged.hpp"

namespace qw {

namespace {

constexpr int kRound = 128;             // keys of a round: 4 waves of 32
constexpr float kNone = -0x1p100f;      // a maximum below every score
constexpr float kLazy = 4.0f;           // scores pass the reference by so much (log2) before it follows
constexpr float kLift = 11.0f;          // log2 of P at the reference: P <= 2^15 fits a half, and 2^-25 of it too

struct AttendArgs {
    PagedView c;
    const f16* q;
    int64_t q_seq, q_head, q_row;
    f16* out;
    const int32_t* lengths;
    const int32_t* table;
    int64_t table_stride;
    int width, n_seq, G, n_rows, R;  // R = G * n_rows rows of a KV head: row g * n_rows + r
    const int32_t* picked;
    int n_picked;
    float scale2;  // scale * log2 e
    int workers;
    float* part_o;    // [workers][2][hkv][R][D]
    float2* part_ml;  // [workers][2][hkv][R]
};

// A sequence's keys as the kernel walks them: the whole of it, or its picked pages side by side.
__device__ __forceinline__ int keys_of(const AttendArgs& a, int b) {
    const int len = min(max(a.lengths[b], 0), a.width << a.c.lg);
    if (!a.picked) return len;
    const int pages = (len + (1 << a.c.lg) - 1) >> a.c.lg;
    return min(pages, a.n_picked) << a.c.lg;
}
__device__ __forceinline__ uint32_t rounds_of(const AttendArgs& a, int b) {
    return (uint32_t)(keys_of(a, b) + kRound - 1) / kRound;
}
__device__ __forceinline__ uint32_t total_rounds(const AttendArgs& a) {
    const int lane = (int)__lane_id();
    uint32_t n = 0;
    for (int b = lane; b < a.n_seq; b += 64) n += rounds_of(a, b);
    return (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(n), 63);
}

// (a round at least for each that works)
__device__ __forceinline__ uint32_t workers_of(const AttendArgs& a, uint64_t total) {
    return (uint64_t)a.workers < total ? (uint32_t)a.workers : (uint32_t)total;
}

// 32 keys' place: of each 16 the pool's page, the slot, and the position of the first; the pages' V exponent.
struct Place {
    int page0, page1, slot0, slot1, pos0, pos1, e0, e1;
};
// Tables, picks and exponents are read by scalar loads: a vector load would wait for the keys requested before it.
typedef const int32_t __attribute__((address_space(4))) * Scalars;
__device__ __forceinline__ Scalars scalars(const int32_t* p) { return (Scalars)(uintptr_t)p; }
constexpr int kNoKey = 0x7fffff00;  // a position behind every key

template <int BITS, int D, bool INT8>
struct Chunk {
    static constexpr int NG = INT8 ? 1 : D / kGroup;
    static constexpr int NK = D * BITS / 512;      // 16-byte pieces of a K row a lane group
    static constexpr int DPP = BITS == 16 ? 1 : 16 / BITS;  // dims of a V piece
    static constexpr int NV = D / 16 / DPP;
    static constexpr int PAR = INT8 ? 8 : 16 * NG;  // halves of 8 keys' scales and biases
    u32x4 k[2][NK];
    u32x4 v[NV];
    half8 ks[NG], kb[NG], vs[NG], vb;
};

template <int BITS, int D, bool INT8>
__device__ __forceinline__ void load_k(Chunk<BITS, D, INT8>& x, const PagedView& c, const Place& p, int h, int lane) {
    using C = Chunk<BITS, D, INT8>;
    const int i = lane & 15, g = lane >> 4;
    const int64_t page = lane & 8 ? p.page1 : p.page0;
    const int slot = (lane & 8 ? p.slot1 : p.slot0) + 8 * (i >> 2 & 1) + (i & 3);
    const char* row = c.k + (((page * c.hkv + h) << c.lg) + slot) * (D * BITS / 8) + 16 * g;
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
        for (int j = 0; j < C::NK; j++) x.k[t][j] = *(const u32x4*)(row + t * 4 * (D * BITS / 8) + 64 * j);
    if constexpr (BITS != 16) {
        const int64_t pg = g & 2 ? p.page1 : p.page0;
        const int blk = ((g & 2 ? p.slot1 : p.slot0) >> 3) + (g & 1);
        const f16* par = c.k_par + (((pg * c.hkv + h) << (c.lg - 3)) + blk) * C::PAR;
#pragma unroll
        for (int m = 0; m < C::NG; m++) {
            x.ks[m] = *(const half8*)(par + 8 * m);
            if (!INT8) x.kb[m] = *(const half8*)(par + 8 * (C::NG + m));
        }
    }
}
template <int BITS, int D, bool INT8>
__device__ __forceinline__ void load_v(Chunk<BITS, D, INT8>& x, const PagedView& c, const Place& p, int h, int lane) {
    using C = Chunk<BITS, D, INT8>;
    const int n = lane & 15, g = lane >> 4;
    const int64_t pg = g & 2 ? p.page1 : p.page0;
    const int64_t blk = (((pg * c.hkv + h) << (c.lg - 3)) + ((g & 2 ? p.slot1 : p.slot0) >> 3) + (g & 1));
    const char* at = c.v + blk * (D * BITS) + 16 * n;
#pragma unroll
    for (int j = 0; j < C::NV; j++) x.v[j] = *(const u32x4*)(at + 256 * j);
    if constexpr (BITS != 16) {
        const f16* par = c.v_par + blk * C::PAR;
#pragma unroll
        for (int m = 0; m < C::NG; m++) x.vs[m] = *(const half8*)(par + 8 * m);
        if (!INT8) x.vb = *(const half8*)(par + 8 * (C::NG + min(n, C::NG - 1)));
    }
}

// 8 codes of a K piece as halves code * 2^-24.
template <int BITS>
__device__ __forceinline__ half8 k_codes(const u32x4* k, int m) {
    if constexpr (BITS == 16) {
        return as_h8(k[m]);
    } else if constexpr (BITS == 8) {
        const uint32_t w0 = k[m / 2][2 * (m & 1)], w1 = k[m / 2][2 * (m & 1) + 1];
        return as_h8(u32x4{__builtin_amdgcn_perm(0u, w0, 0x0C010C00u), __builtin_amdgcn_perm(0u, w0, 0x0C030C02u),
                           __builtin_amdgcn_perm(0u, w1, 0x0C010C00u), __builtin_amdgcn_perm(0u, w1, 0x0C030C02u)});
    } else {
        const uint32_t w = k[m / 4][m & 3], f = 0x000F000Fu;
        return as_h8(u32x4{w & f, w >> 4 & f, w >> 8 & f, w >> 12 & f});
    }
}
// 8 keys' codes of dim e of a V piece; of 4 bits pairs 1 and 3 at 16 times their value.
template <int BITS>
__device__ __forceinline__ half8 v_codes(u32x4 v, int e) {
    if constexpr (BITS == 16) {
        return as_h8(v);
    } else if constexpr (BITS == 8) {
        const uint32_t w0 = v[2 * e], w1 = v[2 * e + 1];
        return as_h8(u32x4{__builtin_amdgcn_perm(0u, w0, 0x0C010C00u), __builtin_amdgcn_perm(0u, w0, 0x0C030C02u),
                           __builtin_amdgcn_perm(0u, w1, 0x0C010C00u), __builtin_amdgcn_perm(0u, w1, 0x0C030C02u)});
    } else {
        const uint32_t w = v[e], w8 = w >> 8;
        return as_h8(u32x4{w & 0x000F000Fu, w & 0x00F000F0u, w8 & 0x000F000Fu, w8 & 0x00F000F0u});
    }
}

__device__ __forceinline__ float4v mfma(half8 a, half8 b, float4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// RT row tiles of 16 in a workgroup, 4 waves each.
template <int BITS, int D, bool INT8, int RT>
__global__ __launch_bounds__(256 * RT, D == 256 ? 2 : 3) void paged_attend_kernel(AttendArgs a) {
    using C = Chunk<BITS, D, INT8>;
    constexpr int NG = C::NG, STEPS = D / 32, DPP = C::DPP;
    extern __shared__ __attribute__((aligned(16))) float lds[];  // [RT][4][rows][D + 4], then (max, sum) [RT][4][16]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int kw = wave & 3, rt = wave >> 2, h = blockIdx.y;
    const int col = lane & 15, g = lane >> 4;
    const int row0 = ((int)blockIdx.z * RT + rt) * 16, rows = max(min(a.R - row0, 16), 0);
    const int tile_rows = min(a.R - (int)blockIdx.z * RT * 16, 16);  // of the workgroup's first tile: the LDS row count

    const uint64_t total = total_rounds(a);
    const uint32_t w = blockIdx.x, workers = workers_of(a, total);
    if (w >= workers) return;
    const uint32_t begin = (uint32_t)(w * total / workers), end = (uint32_t)((w + 1) * total / workers);
    uint32_t at = begin;
    bool first = true;
    while (at < end) {
        const PagedUnit u = find_unit(a.n_seq, at, [&](int b) { return rounds_of(a, b); });
        if (u.b < 0) return;
        const int b = u.b, keys = keys_of(a, b), len = min(max(a.lengths[b], 0), a.width << a.c.lg);
        const uint32_t all = (uint32_t)(keys + kRound - 1) / kRound;
        const uint32_t r0 = u.at, r1 = min(all, u.at + (end - at));
        const Scalars table = scalars(a.table + b * a.table_stride), v_exp = scalars(a.c.v_exp);
        const Scalars picked = scalars(a.picked ? a.picked + ((int64_t)b * a.c.hkv + h) * a.n_picked : nullptr);

        auto half_at = [&](int key, int& page, int& slot, int& pos) {  // (uniform) 16 keys from `key` on
            const int j = key >> a.c.lg;
            slot = key & ((1 << a.c.lg) - 1);
            int logical = key < keys ? (picked ? picked[j] : j) : -1;
            page = (uint32_t)logical < (uint32_t)a.width ? table[logical] : -1;
            const bool there = (uint32_t)page < (uint32_t)a.c.n_pages;
            pos = there ? (logical << a.c.lg) + slot : kNoKey;
            page = there ? page : 0;
        };
        auto place_of = [&](uint32_t r) {
            Place p{};
            if (r >= r1) return p;  // (behind the piece: page 0, which every wave then requests and none uses)
            const int key = (int)(r * kRound) + 32 * kw;
            half_at(key, p.page0, p.slot0, p.pos0);
            half_at(key + 16, p.page1, p.slot1, p.pos1);
            if (BITS != 16) {  // (left as they come: a use here would wait for them)
                p.e0 = v_exp[(int64_t)p.page0 * a.c.hkv + h];
                p.e1 = v_exp[(int64_t)p.page1 * a.c.hkv + h];
            }
            return p;
        };

        // the query rows
        half8 q[STEPS];
        float qsum[NG];
        const int row = row0 + min(col, rows - 1);
        const int rr = row % a.n_rows;
        {
            const f16* qr = a.q + b * a.q_seq + (int64_t)(h * a.G + row / a.n_rows) * a.q_head + rr * a.q_row;
#pragma unroll
            for (int m = 0; m < STEPS; m++) q[m] = rows > 0 ? *(const half8*)(qr + 32 * m + 8 * g) : half8{};
            if constexpr (BITS != 16) {
#pragma unroll
                for (int m = 0; m < NG; m++) {
                    float s = 0.0f;
#pragma unroll
                    for (int j = 0; j < STEPS / NG; j++)
#pragma unroll
                        for (int e = 0; e < 8; e++) s += (float)q[m * (STEPS / NG) + j][e];
                    s += lane_xor<16>(s, lane);
                    s += lane_xor<32>(s, lane);
                    qsum[m] = s * (INT8 ? -128.0f * 0x1p-24f : 0x1p-24f);  // in the codes' units
                }
            }
        }
        const float sc = a.scale2 * (BITS == 16 ? 1.0f : 0x1p24f);
        const int seen = len - a.n_rows + rr + 1;     // keys before it are this row's
        const int seen_all = len - a.n_rows + 1;      // and all rows'

        float4v o[D / 16], ob = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < D / 16; i++) o[i] = float4v{0, 0, 0, 0};
        float M = kNone, l = 0.0f, lp = 0.0f;
        int E = 0;

        C x;
        Place cur = place_of(r0);
        load_k(x, a.c, cur, h, lane);
        load_v(x, a.c, cur, h, lane);
        for (uint32_t r = r0; r < r1; r++) {
            const Place next = place_of(r + 1);
            const int top = max(cur.pos0, cur.pos1) + 15;
            // scores: lane group g has keys 8 g + 4 t + i
            float s[8];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                float4v acc[NG];
#pragma unroll
                for (int m = 0; m < NG; m++) acc[m] = float4v{0, 0, 0, 0};
#pragma unroll
                for (int m = 0; m < STEPS; m++)
                    acc[m / (STEPS / NG)] = mfma(k_codes<BITS>(x.k[t], m), q[m], acc[m / (STEPS / NG)]);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if constexpr (BITS == 16) {
                        float y = acc[0][i];
#pragma unroll
                        for (int m = 1; m < NG; m++) y += acc[m][i];
                        s[4 * t + i] = y;
                    } else if constexpr (INT8) {
                        s[4 * t + i] = (float)x.ks[0][4 * t + i] * (acc[0][i] + qsum[0]);
                    } else {
                        float y = 0.0f;
#pragma unroll
                        for (int m = 0; m < NG; m++) {
                            y = __builtin_fmaf((float)x.ks[m][4 * t + i], acc[m][i], y);
                            y = __builtin_fmaf((float)x.kb[m][4 * t + i], qsum[m], y);
                        }
                        s[4 * t + i] = y;
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            load_k(x, a.c, next, h, lane);
            __builtin_amdgcn_sched_barrier(0);
            const bool masked = top >= seen_all;
#pragma unroll
            for (int i = 0; i < 8; i++) s[i] *= sc;
            if (masked) {
                const int pos = (g & 2 ? cur.pos1 : cur.pos0) + 8 * (g & 1);
#pragma unroll
                for (int i = 0; i < 8; i++) s[i] = pos + i < seen ? s[i] : -INFINITY;
            }
            float mx = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
            if (__any(mx > M + kLazy)) {
                mx = fmaxf(mx, lane_xor<16>(mx, lane));
                mx = fmaxf(mx, lane_xor<32>(mx, lane));
                const float m1 = fmaxf(M, mx), alpha = __builtin_amdgcn_exp2f(M - m1);
                M = m1;
                l *= alpha, lp *= alpha;
                ob *= alpha;
#pragma unroll
                for (int i = 0; i < D / 16; i++) o[i] *= alpha;
            }
            if constexpr (BITS != 16) {
                const int e = max(cur.e0, cur.e1);
                if (e > E) {  // V scales of 1 and more: P gives way, so that P times a scale fits a half
                    const float f = __builtin_amdgcn_exp2f((float)(E - e));
                    E = e;
                    l *= f, lp *= f;
                    ob *= f;
#pragma unroll
                    for (int i = 0; i < D / 16; i++) o[i] *= f;
                }
            }
            const float ref = M + ((float)E - kLift);
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                p[i] = __builtin_amdgcn_exp2f(s[i] - ref);
                l += p[i];
            }
            uint32_t key[4] = {~0u, ~0u, ~0u, ~0u};
            if (masked) {  // what stands behind the sequence's end takes no part, whatever it is
                const int pos = (g & 2 ? cur.pos1 : cur.pos0) + 8 * (g & 1);
#pragma unroll
                for (int j = 0; j < 4; j++) key[j] = (pos + 2 * j < len ? 0xFFFFu : 0u) | (pos + 2 * j + 1 < len ? 0xFFFF0000u : 0u);
            }
            const u32x4 km = {key[0], key[1], key[2], key[3]};
            if constexpr (BITS == 16) {
                half8 ph;
#pragma unroll
                for (int i = 0; i < 8; i++) ph[i] = (f16)p[i];
                if (masked) {
#pragma unroll
                    for (int j = 0; j < C::NV; j++) x.v[j] &= km;
                }
#pragma unroll
                for (int j = 0; j < C::NV; j++) o[j] = mfma(v_codes<16>(x.v[j], 0), ph, o[j]);
            } else {
                if (masked) {
#pragma unroll
                    for (int m = 0; m < NG; m++) x.vs[m] = as_h8(__builtin_bit_cast(u32x4, x.vs[m]) & km);
                    if (!INT8) x.vb = as_h8(__builtin_bit_cast(u32x4, x.vb) & km);
                }
                if constexpr (!INT8) {
                    half8 ph;
#pragma unroll
                    for (int i = 0; i < 8; i++) ph[i] = (f16)p[i];
                    ob = mfma(col < NG ? x.vb : half8{}, ph, ob);
                }
                if constexpr (BITS == 4) p[2] *= 0.0625f, p[3] *= 0.0625f, p[6] *= 0.0625f, p[7] *= 0.0625f;
                constexpr int PER = C::NV / NG;
#pragma unroll
                for (int m = 0; m < NG; m++) {
                    half8 ph;
#pragma unroll
                    for (int i = 0; i < 8; i++) ph[i] = (f16)(p[i] * (float)x.vs[m][i]);
                    if constexpr (INT8) {
#pragma unroll
                        for (int i = 0; i < 8; i++) lp += (float)ph[i];
                    }
#pragma unroll
                    for (int j = m * PER; j < (m + 1) * PER; j++)
#pragma unroll
                        for (int e = 0; e < DPP; e++) o[j * DPP + e] = mfma(v_codes<BITS>(x.v[j], e), ph, o[j * DPP + e]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            load_v(x, a.c, next, h, lane);
            __builtin_amdgcn_sched_barrier(0);
            cur = next;
        }

        // the wave's row: sum over the lane groups, biases, the codes' units
        l += lane_xor<16>(l, lane);
        l += lane_xor<32>(l, lane);
        if constexpr (INT8) {
            lp += lane_xor<16>(lp, lane);
            lp += lane_xor<32>(lp, lane);
        }
        float* so = lds + ((rt * 4 + kw) * tile_rows + col) * (D + 4);
        float2* sml = (float2*)(lds + RT * 4 * tile_rows * (D + 4));
        if (!first) __syncthreads();  // (the last piece's sums are read)
        first = false;
        if (g == 0) sml[(rt * 4 + kw) * 16 + col] = float2{M + (float)E, l};
        float bias[NG];
#pragma unroll
        for (int m = 0; m < NG; m++)
            bias[m] = BITS == 16 ? 0.0f : INT8 ? -128.0f * lp : __shfl(ob[m & 3], col);
        if (col < rows) {
#pragma unroll
            for (int j = 0; j < C::NV; j++) {
                float f[4 * DPP];  // dims DPP (16 j + 4 g) ..
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int e = 0; e < DPP; e++) {
                        const float y = o[j * DPP + e][i];
                        f[i * DPP + e] = BITS == 16 ? y : __builtin_fmaf(y, 0x1p24f, bias[INT8 ? 0 : j / (C::NV / NG)]);
                    }
#pragma unroll
                for (int i = 0; i < DPP; i++)
                    *(float4v*)(so + DPP * (16 * j + 4 * g) + 4 * i) = float4v{f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]};
            }
        }
        __syncthreads();
        // the four waves' rows joined by the tile's 256 threads
        const bool done = r0 == 0 && r1 == all;
        const int slot = 2 * (int)w + (u.at == 0 && at != begin ? 1 : 0);
        for (int i = kw * 64 + lane; i < rows * (D / 4); i += 256) {
            const int c = i / (D / 4), d = i % (D / 4) * 4;
            float2 ml[4];
            float mm = kNone;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                ml[k] = sml[(rt * 4 + k) * 16 + c];
                mm = fmaxf(mm, ml[k].x);
            }
            float4v y = {0, 0, 0, 0};
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float f = __builtin_amdgcn_exp2f(ml[k].x - mm);
                y += f * *(const float4v*)(lds + ((rt * 4 + k) * tile_rows + c) * (D + 4) + d);
                sum = __builtin_fmaf(f, ml[k].y, sum);
            }
            const int64_t rw = row0 + c;
            if (done) {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                const int64_t to = ((b * (int64_t)a.c.hkv + h) * a.R + rw) * D + d;
                *(half4v*)(a.out + to) = half4v{(f16)(y[0] * inv), (f16)(y[1] * inv), (f16)(y[2] * inv), (f16)(y[3] * inv)};
            } else {
                const int64_t to = ((int64_t)slot * a.c.hkv + h) * a.R + rw;
                *(float4v*)(a.part_o + to * D + d) = y;
                if (d == 0) a.part_ml[to] = float2{mm, sum};
            }
        }
        at += r1 - r0;
    }
}

// Joins a row's pieces: grid (rows of all heads, n_seq). A sequence within one worker's run was written
// by it; one without keys is zeros.
template <int D>
__global__ __launch_bounds__(256) void paged_merge_kernel(AttendArgs a) {
    constexpr int TC = D / 4, SG = 256 / TC;
    __shared__ float4v sm_o[256];
    __shared__ float sm_l[SG];
    const int tid = threadIdx.x, b = blockIdx.y, h = (int)blockIdx.x / a.R, row = (int)blockIdx.x % a.R;
    const uint64_t total = total_rounds(a);
    const uint32_t mine = rounds_of(a, b);
    uint32_t base = 0;
    {
        uint32_t n = 0;
        const int lane = tid & 63;
        for (int i = lane; i < b; i += 64) n += rounds_of(a, i);
        base = (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(n), 63);
    }
    const int d = tid % TC * 4, sg = tid / TC;
    f16* to = a.out + ((b * (int64_t)a.c.hkv + h) * a.R + row) * D + d;
    if (mine == 0) {
        if (sg == 0) *(half4v*)to = half4v{};
        return;
    }
    const uint32_t workers = workers_of(a, total);
    auto worker_of = [&](uint64_t x) { return (int)(((x + 1) * workers - 1) / total); };
    const int w0 = worker_of(base), w1 = worker_of(base + mine - 1);
    if (w0 == w1) return;
    // its first piece is the last of its worker's run, unless that begins with it
    const int s0 = (uint32_t)((uint64_t)w0 * total / workers) == base ? 2 * w0 : 2 * w0 + 1;
    auto slot_of = [&](int w) { return ((int64_t)(w == w0 ? s0 : 2 * w) * a.c.hkv + h) * a.R + row; };
    float mm = kNone;
    for (int w = w0 + (tid & 63); w <= w1; w += 64) mm = fmaxf(mm, a.part_ml[slot_of(w)].x);
    mm = wave_reduce(mm, OpMax());
    float4v y = {0, 0, 0, 0};
    float sum = 0.0f;
    for (int w = w0 + sg; w <= w1; w += SG) {
        const int64_t s = slot_of(w);
        const float2 ml = a.part_ml[s];
        const float f = __builtin_amdgcn_exp2f(ml.x - mm);
        y += f * *(const float4v*)(a.part_o + s * D + d);
        sum = __builtin_fmaf(f, ml.y, sum);
    }
    sm_o[tid] = y;
    if (tid % TC == 0) sm_l[sg] = sum;
    __syncthreads();
    if (sg) return;
#pragma unroll
    for (int k = 1; k < SG; k++) {
        y += sm_o[k * TC + tid];
        sum += sm_l[k];
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    *(half4v*)to = half4v{(f16)(y[0] * inv), (f16)(y[1] * inv), (f16)(y[2] * inv), (f16)(y[3] * inv)};
}

template <int BITS, int D, bool INT8, int RT>
int launch_attend(const AttendArgs& a, int groups, hipStream_t stream) {
    const int rows = std::min(a.R, 16);
    const size_t lds = (size_t)RT * 4 * (rows * (D + 4) * 4 + 16 * 8);
    const void* f = (const void*)paged_attend_kernel<BITS, D, INT8, RT>;
    if (int rc = ensure_dynamic_lds(f, lds)) return rc;
    hipLaunchKernelGGL((paged_attend_kernel<BITS, D, INT8, RT>), dim3(a.workers, a.c.hkv, groups), dim3(256 * RT), lds, stream, a);
    QW_HIP_CHECK(hipGetLastError());
    return QW_OK;
}
template <int BITS, bool INT8>
int launch_rows(const AttendArgs& a, int D, hipStream_t stream) {
    const int tiles = (a.R + 15) / 16;
    if (tiles == 1) return D == 256 ? launch_attend<BITS, 256, INT8, 1>(a, 1, stream) : launch_attend<BITS, 128, INT8, 1>(a, 1, stream);
    return D == 256 ? launch_attend<BITS, 256, INT8, 2>(a, (tiles + 1) / 2, stream) : launch_attend<BITS, 128, INT8, 2>(a, (tiles + 1) / 2, stream);
}

}  // namespace

int check_query(const PagedCache& c, const PagedQuery& q, const char* what) {
    const std::string w(what);
    QW_REQUIRE(q.n_seq >= 0 && q.n_seq <= 65535 && q.n_rows > 0 && q.n_q_heads > 0 && q.n_q_heads % c.hkv == 0,
               QW_ERR_INVALID_ARGUMENT, w + ": 0 .. 65535 sequences, n_rows > 0 and n_q_heads a multiple of the KV heads expected");
    QW_REQUIRE(q.n_seq == 0 || (q.q && q.lengths && (q.table || q.table_width == 0)), QW_ERR_INVALID_ARGUMENT, w + ": null q/lengths/table");
    QW_REQUIRE(q.table_width >= 0 && q.table_stride >= q.table_width && (int64_t)q.table_width * c.page_size <= 0x7fffff00,
               QW_ERR_INVALID_ARGUMENT, w + ": table_width >= 0, not above its stride, and table_width * page_size < 2^31 expected");
    QW_REQUIRE((uintptr_t)q.q % 16 == 0 && (q.seq_stride | q.head_stride | q.row_stride) % 8 == 0 && q.seq_stride >= 0 &&
                   q.head_stride >= 0 && q.row_stride >= 0,
               QW_ERR_INVALID_ARGUMENT, w + ": q 16-byte aligned with strides of whole 16 bytes expected");
    const int64_t rows = (int64_t)(q.n_q_heads / c.hkv) * q.n_rows;
    QW_REQUIRE(rows <= 16384 && rows * c.hkv <= (1 << 22), QW_ERR_UNSUPPORTED, w + ": at most 16384 query rows a KV head");
    return QW_OK;
}

int paged_attention(PagedCache& c, const PagedQuery& q, const int32_t* picked, int n_picked, float scale, void* out,
                    hipStream_t stream) {
    if (int rc = check_query(c, q, "paged attention")) return rc;
    QW_REQUIRE(scale >= -0x1p40f && scale <= 0x1p40f, QW_ERR_INVALID_ARGUMENT, "paged attention: |scale| <= 2^40 expected");
    QW_REQUIRE(!picked || (n_picked > 0 && (int64_t)n_picked * c.page_size <= 0x7fffff00), QW_ERR_INVALID_ARGUMENT,
               "paged attention: n_picked > 0 with n_picked * page_size < 2^31 expected");
    if (q.n_seq == 0) return QW_OK;
    QW_REQUIRE(out && (uintptr_t)out % 8 == 0, QW_ERR_INVALID_ARGUMENT, "paged attention: out null or off 8 bytes");
    const int64_t most = std::min<int64_t>(q.table_width, picked ? n_picked : q.table_width) * c.page_size;  // keys of a sequence
    const int64_t rounds = (most + kRound - 1) / kRound * q.n_seq;
    QW_REQUIRE(rounds < (1ll << 31), QW_ERR_UNSUPPORTED, "paged attention: n_seq * table_width * page_size below 2^38 expected");
    // (one handle, a stream a thread: they would share a workspace)
    QW_REQUIRE(stream != hipStreamPerThread, QW_ERR_UNSUPPORTED, "paged attention: hipStreamPerThread; name a stream");
    DeviceGuard dg(c.device);
    QW_REQUIRE(dg.ok, QW_ERR_HIP, "paged attention: hipSetDevice failed");
    AttendArgs a{};
    a.c = c.view;
    a.q = (const f16*)q.q;
    a.q_seq = q.seq_stride, a.q_head = q.head_stride, a.q_row = q.row_stride;
    a.out = (f16*)out;
    a.lengths = q.lengths;
    a.table = q.table;
    a.table_stride = q.table_stride;
    a.width = q.table_width;
    a.n_seq = q.n_seq;
    a.G = q.n_q_heads / c.hkv;
    a.n_rows = q.n_rows;
    a.R = a.G * q.n_rows;
    a.picked = picked;
    a.n_picked = n_picked;
    a.scale2 = scale * kLog2e;
    const int groups = a.R <= 16 ? 1 : ((a.R + 15) / 16 + 1) / 2;
    a.workers = (int)std::max<int64_t>(1, std::min<int64_t>(rounds, 512 / ((int64_t)c.hkv * groups)));
    const int64_t parts = (int64_t)a.workers * 2 * c.hkv * a.R;
    void* ws = nullptr;
    if (int rc = workspace(kWsPaged, c.device, stream, (size_t)(parts * (c.D * 4 + 8)), &ws)) return rc;
    a.part_o = (float*)ws;
    a.part_ml = (float2*)(a.part_o + parts * c.D);
    if (rounds > 0) {
        const int rc = c.bits == 16 ? launch_rows<16, false>(a, c.D, stream)
                       : c.bits == 4 ? launch_rows<4, false>(a, c.D, stream)
                       : c.int8()    ? launch_rows<8, true>(a, c.D, stream)
                                     : launch_rows<8, false>(a, c.D, stream);
        if (rc) return rc;
    }
    const dim3 grid((unsigned)(c.hkv * a.R), q.n_seq);
    if (c.D == 256)
        hipLaunchKernelGGL(paged_merge_kernel<256>, grid, dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL(paged_merge_kernel<128>, grid, dim3(256), 0, stream, a);
    QW_HIP_CHECK(hipGetLastError());
    return QW_OK;
}

}  // namespace qw
