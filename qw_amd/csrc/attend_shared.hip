// attend_shared.hip - attention of many sequences' rows over a cache that they
// share and a cache of their own parts, gfx950.
//
// For row r (of Tq) of sequence b, query head j of KV head h, with x = scale q:
//   out = sum_t p_t v_t,  p = softmax over t of x . k_t,
// t over every key of the prefix cache's head h and over keys starts[b] ..
// T_tail - Tq + r of the tail cache's head b * hkv + h. The runtime's own path
// for it would be one cache a sequence, each with the prefix in it
// (KVCache::update_and_turbo4_causal_attention, crates/mlxcel-core/src/
// cache.rs:3520): n_seq reads of the prefix where this makes one.
//
// The softmax is associative in blocks: a set of keys is summed up by m = max
// s_t, l = sum e^(s_t - m), O = sum e^(s_t - m) v_t, and two sets join as
// (max(m, m'), l e^(m-M) + l' e^(m'-M), O e^(m-M) + O' e^(m'-M)). So the
// prefix, whose keys all rows of a KV head see (n_seq Tq G of them), and the
// tails, each seen by Tq G rows, are units of one launch (of one each where the
// caches' widths differ), both cut into key splits, and a merge launch joins the
// partials. The splits are those of the least estimated time on 256 CUs
// (plan_shared).
//
// Two kernels, by the rows of a unit: many_body up to 128 (D = 256) or 256 rows
// over key tiles in LDS, dequantized beside the MFMAs by waves of their own;
// few_body up to 16, which have nothing to share and read keys straight into MFMA
// operands. Many query tiles over one quantized cache read images of its tiles,
// dequantized once (kImageQueryTiles).
// Rounded to fewer than 32 bits: P, to fp16 (a weight by at most 2^-11 of itself, below
// 2^-14 by 2^-25, averaged over the keys; the output's own rounding is the larger), the
// output, and over Turbo4 caches the rotated q and output.
//
// Whole calls against their floors (the keys once at 4.98 TB/s, the products at 1.15 PFLOP/s): 16
// sequences over 32k 4-bit keys 34.2 us of 11.3, 64 over 64k fp16 keys 105 of 61.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <initializer_list>
#include <type_traits>

#include "attend_shared.hpp"
#include "block_tile.hpp"
#include "dequant.hpp"
#include "kv_cache.hpp"
#include "turbo4_device.hpp"

namespace qw {

namespace {

constexpr int kWaves = 8, kFillWaves = 4;
// Query tiles from which the key tiles of one quantized cache are laid out once. 256-row tiles of 8 heads,
// D = 128, and 128-row ones of 4, D = 256, over 4k, 9.7k and 32k 4-bit, 8-bit and Int8 keys, dequantized in each /
// laid out: 8 tiles slower laid out by 0 to 8 %, 12 tiles 7 % faster to 5 % slower (32k 4-bit keys 420 / 416 and 229 /
// 229 us), 16 tiles 6 % faster to 2 % slower (514 / 494, 293 / 286), 20 faster but for Int8 at D = 128 (109 / 115 at 4k),
// 44 by 2 to 18 % (1461 / 1329, 813 / 748).
constexpr int kImageQueryTiles = 16;
constexpr int kFewRows = 16;  // of a unit of the kernel for few rows
// 16-row tiles a computing wave of the other, in 168 registers (three waves a SIMD). 4- and 8-bit instances spill one
// at most, but fp16 and Turbo4 ones, whose filling waves stage more, 12 to 17.
__host__ __device__ constexpr int many_tiles(int D) { return D == 256 ? 1 : 2; }

// A unit: a split of a query tile of a head of one of the two caches.
struct Unit {
    int sp, hc, h, row_base;      // split; the cache's head, the KV head; the head's first row of the KV head's R
    int row0, row_end;            // the unit's rows
    int lo, hi;                   // keys that any of them sees
    int k_begin, k_end;           // the split's keys
    int T, cap, causal_rows;
    int64_t slot_base;            // partial rows: slot_base + row
    uint32_t code_off;
    const uint32_t *k_data, *k_params, *v_data, *v_params;
    __device__ int limit(int row, int G) const {  // a row's last visible key
        return causal_rows ? T - causal_rows + (row - row_base) / G : T - 1;
    }
};
template <int D>
__device__ __forceinline__ Unit this_unit(const SharedArgs& a) {
    const bool tail = (int)blockIdx.x >= a.seg[0].n_units;
    const int id = (int)blockIdx.x - (tail ? a.seg[0].n_units : 0);
#define QW_SEG(f) (tail ? a.seg[1].f : a.seg[0].f)
    Unit u;
    const int n_split = QW_SEG(n_split), heads = QW_SEG(heads), rows = QW_SEG(rows), unit_rows = QW_SEG(unit_rows);
    const int qt = id / n_split / heads;
    u.sp = id % n_split;
    u.hc = id / n_split % heads;
    u.h = u.hc % a.hkv;
    u.row_base = u.hc / a.hkv * rows;
    u.row0 = u.row_base + qt * unit_rows;
    u.row_end = u.row_base + min(rows, (qt + 1) * unit_rows);
    u.T = QW_SEG(T);
    u.cap = QW_SEG(cap);
    u.causal_rows = QW_SEG(causal_rows);
    u.lo = tail && a.starts ? min(max(a.starts[u.hc / a.hkv], 0), u.T) : 0;
    u.hi = u.limit(u.row_end - 1, a.G) + 1;
    const int tile = shared_tile(D), keys = QW_SEG(tiles_per_split) * tile;
    u.k_begin = u.lo / tile * tile + u.sp * keys;
    u.k_end = min(u.hi, u.k_begin + keys);
    u.slot_base = ((int64_t)(QW_SEG(slot0) + u.sp) * a.hkv + u.h) * a.R;
    u.code_off = QW_SEG(code_off2);
    u.k_data = QW_SEG(k_data);
    u.k_params = QW_SEG(k_params);
    u.v_data = QW_SEG(v_data);
    u.v_params = QW_SEG(v_params);
#undef QW_SEG
    return u;
}
// Row `row` of KV head h: its place in q and out, in rows of D.
__device__ __forceinline__ int64_t q_row(const SharedArgs& a, int h, int row) {
    const int seq = row / (a.Tq * a.G), x = row % (a.Tq * a.G);
    return ((int64_t)seq * a.hkv * a.G + h * a.G + x % a.G) * a.Tq + x / a.G;
}
// 16 bytes of q as the kernels take them: negated where the scale is negative, and for 4-bit
// codes in the order in which deq4 leaves a word's dims, (0,4), (1,5), (2,6), (3,7).
template <int KIND>
__device__ __forceinline__ u32x4 q_piece(u32x4 w, uint32_t flip) {
    w ^= u32x4{flip, flip, flip, flip};
    if constexpr (KIND == 4)
        w = u32x4{__builtin_amdgcn_perm(w.z, w.x, 0x05040100u), __builtin_amdgcn_perm(w.z, w.x, 0x07060302u),
                  __builtin_amdgcn_perm(w.w, w.y, 0x05040100u), __builtin_amdgcn_perm(w.w, w.y, 0x07060302u)};
    return w;
}

// Schedules a run of N LDS reads that each feed MF MFMAs with four reads kept ahead of them (left to
// itself the compiler waits for each).
template <int GROUP, int N, int MF>
__device__ __forceinline__ void keep_reads_ahead() {
    constexpr int AH = 4;
    __builtin_amdgcn_sched_group_barrier(0x100, AH, GROUP);
#pragma unroll
    for (int i = 0; i < N - AH; i++) {
        __builtin_amdgcn_sched_group_barrier(0x008, MF, GROUP);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, GROUP);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, MF * AH, GROUP);
}

// A dequantizing group of 256 threads: a key tile's codes through registers into an LDS tile of
// block_tile.hpp's layout, V's slots in the fp16 order whatever the codes'. The values are
// f16(f16(code * scale) + bias), as the fetch gives them. NATURAL: K's dims in order also from 4-bit
// codes (else pairs (0,4), (1,5), (2,6), (3,7) of each eight). T4: a Turbo4 cache's 4-bit indices, K
// and V row-major, a word a row beside them; cp: the pair of centroids of every byte of them, in LDS.
template <int KIND, int D, bool FAST, bool NATURAL, bool T4 = false>
struct TileFiller {
    using S = BlockShape<D>;
    static constexpr int KT = S::KT, TPR = S::TPR, TPB = S::TPB, NG = S::NG, DPL = D / 16;
    static constexpr int PER = KT * TPR / (64 * kFillWaves);  // slices of each kind a thread
    static constexpr int KU = KIND / 4;                       // 16-byte loads of a 32-dim K slice / 4-slot V slice
    static_assert(PER * 64 * kFillWaves == KT * TPR && (KT / 8) * TPB == KT * TPR, "whole slices a thread");
    struct Stage {
        u32x4 kc[PER][KU], vc[PER][KU], vp[PER][2];
        uint32_t kp[PER];
        uint32_t vt[T4 ? PER : 1][8];  // 4 dims of the 8 rows
    };
    const char *k_head, *kp_head, *v_head, *vp_head;
    // slice j: key kk's 32 dims from 32 q32, V block vb's 4 slots from 4 vj
    int q32[PER], kk[PER], vb[PER], vj[PER];
    uint32_t code_off, magic;
    // key0: the first key of tile 0 of head hc; t: the thread's place in the group
    __device__ TileFiller(const SharedSegment& c, int hc, int key0, int t) {
        const int64_t row = (int64_t)hc * c.cap + key0;
        k_head = (const char*)c.k_data + row * (D * KIND / 8);
        kp_head = (const char*)c.k_params + row * (T4 ? 4 : NG * 4);
        v_head = (const char*)c.v_data + row / 8 * (D * KIND);
        vp_head = (const char*)c.v_params + row / 8 * (T4 ? 32 : NG * 32);
        code_off = c.code_off2;
        magic = vconst(kMagic);
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int x = t + 64 * kFillWaves * j;
            q32[j] = (x >> 4) & (TPR - 1);
            kk[j] = (x & 15) | ((x >> (4 + S::LTPR)) << 4);
            vb[j] = x / TPB;
            vj[j] = x % TPB;
        }
    }
    __device__ __forceinline__ int v_n(int j) const {  // lane group of slot 4 vj
        return KIND == 16 ? 0 : KIND == 8 ? (2 * vj[j]) % 16 : vj[j] % 16;
    }
    __device__ __forceinline__ void load(Stage& st, int i) const {
        const int64_t key = (int64_t)i * KT;
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const u32x4* k = (const u32x4*)(k_head + key * (D * KIND / 8) + (kk[j] * (D * KIND / 8) + 16 * KU * q32[j]));
            const u32x4* v = (const u32x4*)(v_head + key / 8 * (D * KIND) + (vb[j] * (D * KIND) + 16 * KU * vj[j]));
#pragma unroll
            for (int x = 0; x < KU; x++) st.kc[j][x] = k[x];
            if constexpr (T4) {
                st.kp[j] = *(const uint32_t*)(kp_head + key * 4 + 4 * kk[j]);
#pragma unroll
                for (int i = 0; i < 8; i++)
                    st.vt[j][i] = *(const uint16_t*)(v_head + key * (D / 2) + ((8 * vb[j] + i) * (D / 2) + 2 * vj[j]));
                const u32x4* p = (const u32x4*)(vp_head + key * 4 + 32 * vb[j]);
                st.vp[j][0] = p[0];
                st.vp[j][1] = p[1];
                continue;
            }
#pragma unroll
            for (int x = 0; x < KU; x++) st.vc[j][x] = v[x];
            if constexpr (KIND != 16) {
                st.kp[j] = *(const uint32_t*)(kp_head + key * (NG * 4) + (kk[j] * (NG * 4) + 4 * k_param_slot(q32[j] >> 1, NG)));
                const u32x4* p = (const u32x4*)(vp_head + key / 8 * (NG * 32) + (vb[j] * (NG * 32) + v_n(j) * DPL / kGroup * 32));
                st.vp[j][0] = p[0];
                st.vp[j][1] = p[1];
            }
        }
    }
    // The tile whose first key is key0; keys outside [lo, hi), which no row sees, go in as zeros of V:
    // they have weight 0, but 0 x inf is NaN.
    __device__ __forceinline__ void store(const Stage& st, char* buf, int key0, int lo, int hi, const float2* cp = nullptr) const {
        const bool edge = key0 < lo || key0 + KT > hi;
        half8* const sK = (half8*)buf;
        half8* const sV = (half8*)(buf + S::KBUF);
#pragma unroll
        for (int j = 0; j < PER; j++) {
            half8* const kdst = sK + kaddr<KT>(kk[j], 4 * q32[j]);
            half8 y[4];
            if constexpr (KIND == 16) {
#pragma unroll
                for (int w = 0; w < 4; w++) kdst[w * KT] = as_h8(st.kc[j][w]);
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] = as_h8(st.vc[j][e]);
            } else if constexpr (T4) {
                const float kr = (float)h2(st.kp[j]).x;
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    half8 x;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float2 c = cp[st.kc[j][0][w] >> (8 * i) & 0xFFu];
                        x[2 * i] = t4_f16_product(c.x, kr);
                        x[2 * i + 1] = t4_f16_product(c.y, kr);
                    }
                    kdst[w * KT] = x;
                }
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float vr = (float)h2(st.vp[j][i / 4][i % 4]).y;
                    const float2 c0 = cp[st.vt[j][i] & 0xFFu], c1 = cp[st.vt[j][i] >> 8];
                    y[0][i] = t4_f16_product(c0.x, vr);
                    y[1][i] = t4_f16_product(c0.y, vr);
                    y[2][i] = t4_f16_product(c1.x, vr);
                    y[3][i] = t4_f16_product(c1.y, vr);
                }
            } else {
                const half2v sb = h2(st.kp[j]), s = {sb.x, sb.x}, b = {sb.y, sb.y};
                const PairConsts kc = make_consts<FAST, KIND>(s, s, s, s, b, b, b, b, code_off);
                const u32x4 vs = st.vp[j][0], vo = st.vp[j][1];
                const PairConsts vc = make_consts<FAST, KIND>(h2(vs[0]), h2(vs[1]), h2(vs[2]), h2(vs[3]), h2(vo[0]), h2(vo[1]),
                                                              h2(vo[2]), h2(vo[3]), code_off);
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    if constexpr (KIND == 4) {
                        u32x4 x = __builtin_bit_cast(u32x4, deq4<FAST>(st.kc[j][0][w], kc, magic));
                        if constexpr (NATURAL)
                            x = u32x4{__builtin_amdgcn_perm(x.y, x.x, 0x05040100u), __builtin_amdgcn_perm(x.w, x.z, 0x05040100u),
                                      __builtin_amdgcn_perm(x.y, x.x, 0x07060302u), __builtin_amdgcn_perm(x.w, x.z, 0x07060302u)};
                        kdst[w * KT] = as_h8(x);
                        y[w] = deq4<FAST>(st.vc[j][0][w], vc, magic);
                    } else {
                        kdst[w * KT] = deq8<FAST>(st.kc[j][KU / 2 * (w / 2)][2 * (w % 2)], st.kc[j][KU / 2 * (w / 2)][2 * (w % 2) + 1], kc);
                        y[w] = deq8<FAST>(st.vc[j][KU / 2 * (w / 2)][2 * (w % 2)], st.vc[j][KU / 2 * (w / 2)][2 * (w % 2) + 1], vc);
                    }
                }
            }
            if (edge) {
                asm volatile("");
                const int key = key0 + 8 * vb[j];
                const u32x4 keep = keep_keys(hi - key) & ~keep_keys(lo - key);
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] = as_h8(__builtin_bit_cast(u32x4, y[e]) & keep);
            }
            const int vr = KIND == 8 ? 2 * (vj[j] / 8) : 4 * (vj[j] / 16);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int at = T4           ? 17 * ((4 * vj[j] + e) % DPL) + (4 * vj[j] + e) / DPL
                               : KIND == 16 ? 4 * vj[j] + e + (vj[j] >> 2)
                               : KIND == 8 ? 17 * (vr + e % 2) + v_n(j) + e / 2
                                           : 17 * (vr + e) + v_n(j);
                sV[vb[j] * S::VROW + at] = y[e];
            }
        }
    }
};

// Units of many rows, 12 waves. Waves 8 to 11, one a SIMD, dequantize: tile i + 1 (its codes in
// registers since two tiles ago) into the free one of two LDS buffers, then request tile i + 3's codes;
// IMAGE: they copy tile i + 1 from images of the tiles that a launch before made once. Waves 0 to 7, two a
// SIMD, compute tile i, RT row tiles of 16 each:
//   S^T = K . Q^T (a lane then holds 8 consecutive keys of a row, the A operand of P . V), scores in
//   fp32, P in fp16 against a reference that moves when a score passes it by kLazy = 8 powers of two
//   (fp16 keeps 11 bits of p up to 2^8 as well; the accumulators are rescaled in few tiles),
//   O += P . V in fp32.
// Where the rows leave waves free these take parts of each tile's keys, joined at the end through LDS.
// fp16: of K there is no such prefetch. Its loads compile to flat ones, which an LDS wait, so the one before each
// tile's barrier, waits for, and the spilled registers are two of a thread's eight staged pieces, each waited for
// behind its load.
// One barrier a tile. (With 8 waves that dequantize and compute in turn, all of them were in the same
// phase: LDS idle while they dequantize, the VALU while they read: 126 rows over 32k 8-bit keys, D =
// 256, 42 against 38.4 us.)
// Bound by filling and computing at once, which share the VALU and LDS: 96 rows over 131k 4-bit keys, D =
// 256, take 89 us with their merge; the filling waves alone 66, the computing ones alone 75; 8-bit 96, 77 and
// 76; fp16 139, 136 and 78 (filling reads the keys' 537 MB at 4.1 TB/s); all nine with the partials' stores
// some 6 us longer than part_dim's order has them. 16 sequences over 32k 4-bit keys take 31 us, 6 of them
// without any tile or partial, and the merge 5.
// Turbo4: a byte's two centroids come from a table in LDS, four reads a word where the affine modes have a
// few VALU instructions: 16 sequences over 32k keys 58 us with the rotations, 41 over 4-bit codes.
template <int KIND, int D, bool FAST, bool IMAGE, bool T4 = false>
__device__ __forceinline__ void many_body(const SharedArgs& a, char* lds) {
    using S = BlockShape<D>;
    constexpr int KT = S::KT, NSUB = S::NSUB, NM = S::NM, NT = S::NT, VROW = S::VROW, BUF = S::BUF, KBUF = S::KBUF;
    constexpr int RT = many_tiles(D);
    constexpr float kLazy = 8.0f;
    static_assert(2 * BUF <= kSharedLds, "LDS");
    const Unit u = this_unit<D>(a);
    const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = max(0, (u.k_end - u.k_begin + KT - 1) / KT);  // tiles
    const int n_rt = (u.row_end - u.row0 + 16 * RT - 1) / (16 * RT);  // a computing wave each
    // Wave w computes row tile rt_i, its part of each tile's keys; a part above 0 parks its sums in region
    // w - park0 and part 0 joins them, dist waves apart. Five or six row tiles would leave two SIMDs
    // (w mod 4) twice the work of the others: waves 4 to 7 then take halves of the last two.
    const bool halves = RT == 1 && NSUB == 2 && (n_rt == 5 || n_rt == 6);
    const int lrt = n_rt <= 1 ? 0 : n_rt <= 2 ? 1 : n_rt <= 4 ? 2 : 3;
    const int parts = halves ? (wave < 4 ? 1 : 2) : min(kWaves >> lrt, NSUB);
    const int dist = halves ? 2 : 1 << lrt, park0 = halves ? 6 : dist;
    const int rt_i = !halves ? wave & (dist - 1) : wave < 4 ? wave : 4 + (wave & 1);
    const int part = !halves ? wave >> lrt : wave < 4 ? 0 : wave >> 1 & 1;
    const bool joined = halves || parts > 1;  // (the same in all waves)
    constexpr int REG = RT * (64 * NT * 16 + 64 * 8);  // a parked part
    static_assert((kWaves - kWaves / (NSUB < 8 ? NSUB : 8)) * REG <= kSharedLds, "the parked parts fit");

    float2* const cp = (float2*)(lds + 2 * BUF);  // T4: a byte's two centroids
    if constexpr (T4) {
        static_assert(2 * BUF + 256 * sizeof(float2) <= kSharedLds, "the centroid pairs behind the tiles");
        const float* const cb = (int)blockIdx.x >= a.seg[0].n_units ? a.seg[1].t4_cb : a.seg[0].t4_cb;
        for (int i = tid; i < 256; i += 64 * (kWaves + kFillWaves)) cp[i] = float2{cb[i & 15], cb[i >> 4]};
        __syncthreads();
    }
    if (wave >= kWaves) {
        // ---- filling waves
        const SharedSegment& seg = (int)blockIdx.x >= a.seg[0].n_units ? a.seg[1] : a.seg[0];
        if constexpr (IMAGE) {
            // tile i's image into its buffer by LDS-DMA, 1 KB a wave instruction; M0, which gives its place
            // in LDS, is saved and restored so that the compiler's view of it holds
            const char* const img = seg.images + ((int64_t)u.hc * seg.n_tiles + u.k_begin / KT) * BUF + 16 * lane;
            const uint32_t lds0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)lds;
            static_assert(BUF % 1024 == 0, "whole DMA instructions");
            auto copy = [&](int i) {
                for (int c = wave - kWaves; c < BUF / 1024; c += kFillWaves) {
                    uint32_t saved;
                    asm volatile(
                        "s_mov_b32 %0, m0\n\t"
                        "s_mov_b32 m0, %2\n\t"
                        "s_nop 0\n\t"
                        "global_load_lds_dwordx4 %1, off\n\t"
                        "s_nop 0\n\t"
                        "s_mov_b32 m0, %0"
                        : "=&s"(saved)
                        : "v"(img + (int64_t)i * BUF + 1024 * c),
                          "s"(__builtin_amdgcn_readfirstlane(lds0 + BUF * (i & 1) + 1024 * c))
                        : "memory");
                }
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            };
            if (n > 0) copy(0);
            __syncthreads();
            for (int i = 0; i < n; i++) {
                if (i + 1 < n) copy(i + 1);
                __syncthreads();
            }
        } else {
            using Filler = TileFiller<KIND, D, FAST, false, T4>;
            const Filler f(seg, u.hc, u.k_begin, tid - 64 * kWaves);
            auto put = [&](const typename Filler::Stage& st, int i) {
                f.store(st, lds + BUF * (i & 1), u.k_begin + i * KT, u.lo, u.hi, cp);
            };
            typename Filler::Stage s0, s1;  // tiles 1, 3, .. and 2, 4, ..
            if (n > 0) {
                f.load(s0, 0);
                if (n > 2) f.load(s1, 2);
                put(s0, 0);
                if (n > 1) f.load(s0, 1);
            }
            __syncthreads();
            for (int i = 0; i < n; i += 2) {
                if (i + 1 < n) {
                    put(s0, i + 1);
                    if (i + 3 < n) f.load(s0, i + 3);
                }
                __syncthreads();
                if (i + 1 >= n) break;
                if (i + 2 < n) {
                    put(s1, i + 2);
                    if (i + 4 < n) f.load(s1, i + 4);
                }
                __syncthreads();
            }
        }
        if (joined) __syncthreads();
        return;
    }

    // ---- computing waves: RT row tiles, and a part of each tile's keys
    const int wrow0 = u.row0 + 16 * RT * rt_i;
    const bool live = part < parts && wrow0 < u.row_end;
    const int wave_first_lim = u.limit(min(wrow0, u.row_end - 1), a.G), wave_lim = u.limit(min(wrow0 + 16 * RT - 1, u.row_end - 1), a.G);
    int lim[RT];
    half8 qb[RT][NM];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const int row = wrow0 + 16 * rt + r16;
        const bool ok = live && row < u.row_end;
        lim[rt] = ok ? u.limit(row, a.G) : -1;
        const f16* q = a.q + q_row(a, u.h, ok ? row : u.row0) * D + 8 * g;
#pragma unroll
        for (int m = 0; m < NM; m++) {
            const u32x4 w = *(const u32x4*)(q + 32 * m);
            qb[rt][m] = as_h8(q_piece<T4 ? 16 : KIND>(ok ? w : u32x4{0, 0, 0, 0}, a.q_flip));
        }
    }
    float m_ref[RT], l_run[RT];  // log2 units; l: this lane's share
    float4v acc_o[RT][NT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        m_ref[rt] = -INFINITY;
        l_run[rt] = 0.0f;
#pragma unroll
        for (int mm = 0; mm < NT; mm++) acc_o[rt][mm] = float4v{0.f, 0.f, 0.f, 0.f};
    }
    // 32 keys: sub-block ub of tile i
    auto step = [&](int i, int ub) {
        const half8* const sK = (const half8*)(lds + BUF * (i & 1)) + 32 * ub;
        const half8* const sV = (const half8*)(lds + BUF * (i & 1) + KBUF) + (4 * ub + g) * VROW + r16;
        const int key0 = u.k_begin + i * KT + 32 * ub;
        const int kr = 8 * (r16 >> 2) + (r16 & 3), b4 = (kr >> 4) & 1;
        const half8* const k0 = sK + g * KT + kr + 4 * b4;
        const half8* const k1 = sK + g * KT + kr + 4 * (b4 ^ 1);
        float4v s[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; rt++) s[rt][0] = s[rt][1] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int m = 0; m < NM; m++) {
            const half8 x0 = k0[4 * m * KT], x1 = k1[4 * m * KT];
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
                s[rt][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x0, qb[rt][m], s[rt][0], 0, 0, 0);
                s[rt][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x1, qb[rt][m], s[rt][1], 0, 0, 0);
            }
        }
        keep_reads_ahead<0, 2 * NM, RT>();
        if (key0 + 31 > wave_first_lim || key0 < u.lo) {
            asm volatile("");  // a branch, not selects in every step
#pragma unroll
            for (int rt = 0; rt < RT; rt++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int key = key0 + 8 * g + e;
                    if (key > lim[rt] || key < u.lo) s[rt][e >> 2][e & 3] = -INFINITY;
                }
        }
        half8 p16[RT];
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            float mx = s[rt][0][0];
#pragma unroll
            for (int e = 1; e < 8; e++) mx = fmaxf(mx, s[rt][e >> 2][e & 3]);
            mx *= a.scale2;
            if (__any(mx > m_ref[rt] + kLazy)) {
                const float m_new = fmaxf(m_ref[rt], wave_max_g(mx));
                const float alpha = m_ref[rt] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_ref[rt] - m_new);
                l_run[rt] *= alpha;
                float f[4];
#pragma unroll
                for (int e = 0; e < 4; e++) f[e] = __shfl(alpha, 4 * g + e);
#pragma unroll
                for (int mm = 0; mm < NT; mm++)
#pragma unroll
                    for (int e = 0; e < 4; e++) acc_o[rt][mm][e] *= f[e];
                m_ref[rt] = m_new;
            }
            const float ref = m_ref[rt] == -INFINITY ? 0.0f : -m_ref[rt];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rt][e >> 2][e & 3], a.scale2, ref));
                l_run[rt] += p;
                p16[rt][e] = (f16)p;
            }
        }
#pragma unroll
        for (int mm = 0; mm < NT; mm++) {
            const half8 x = sV[17 * mm];
#pragma unroll
            for (int rt = 0; rt < RT; rt++)
                acc_o[rt][mm] = __builtin_amdgcn_mfma_f32_16x16x32_f16(p16[rt], x, acc_o[rt][mm], 0, 0, 0);
        }
        keep_reads_ahead<1, NT, RT>();
    };
    const int per = NSUB / parts, ub0 = part * per;
    __syncthreads();
    for (int i = 0; i < n; i++) {
        if (live)
            for (int ub = ub0; ub < ub0 + per; ub++)
                if (u.k_begin + i * KT + 32 * ub <= wave_lim) step(i, ub);
        __syncthreads();
    }
    // ---- the parts of a wave's rows joined in its part 0, through LDS
    float l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) l[rt] = wave_sum_g(l_run[rt]);
    if (joined) {
        if (live && part > 0) {
            char* reg = lds + (wave - park0) * REG;
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
#pragma unroll
                for (int mm = 0; mm < NT; mm++) ((float4v*)reg)[(rt * NT + mm) * 64 + lane] = acc_o[rt][mm];
                ((float2*)(reg + RT * NT * 64 * 16))[rt * 64 + lane] = float2{m_ref[rt], l[rt]};
            }
        }
        __syncthreads();
        if (live && part == 0) {
            for (int p = 1; p < parts; p++) {
                const char* reg = lds + (wave + p * dist - park0) * REG;
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
                    const float2 ml = ((const float2*)(reg + RT * NT * 64 * 16))[rt * 64 + lane];
                    const float M = fmaxf(m_ref[rt], ml.x), mr = M == -INFINITY ? 0.0f : M;
                    const float fa = __builtin_amdgcn_exp2f(m_ref[rt] - mr), fb = __builtin_amdgcn_exp2f(ml.x - mr);
                    l[rt] = l[rt] * fa + ml.y * fb;
                    m_ref[rt] = M;
                    float xa[4], xb[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        xa[e] = __shfl(fa, 4 * g + e);
                        xb[e] = __shfl(fb, 4 * g + e);
                    }
#pragma unroll
                    for (int mm = 0; mm < NT; mm++) {
                        const float4v o = ((const float4v*)reg)[(rt * NT + mm) * 64 + lane];
#pragma unroll
                        for (int e = 0; e < 4; e++) acc_o[rt][mm][e] = acc_o[rt][mm][e] * xa[e] + o[e] * xb[e];
                    }
                }
            }
        }
    }
    if (!live || part > 0) return;
    // ---- rows out: lane (g, r16) holds dims NT r16 .. + NT - 1 of rows 16 rt + 4 g + e
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        if (g == 0 && wrow0 + 16 * rt + r16 < u.row_end)
            a.part_ml[u.slot_base + wrow0 + 16 * rt + r16] = float2{m_ref[rt], l[rt]};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int row = wrow0 + 16 * rt + 4 * g + e;
            const float le = __shfl(l[rt], 4 * g + e);
            if (row >= u.row_end) continue;
            if (a.n_slots == 1) {
                const float inv = le == 0.0f ? 0.0f : 1.0f / le;
                f16* o = a.out + q_row(a, u.h, row) * D + NT * r16;
#pragma unroll
                for (int c = 0; c < NT; c += 8) {
                    half8 y;
#pragma unroll
                    for (int j = 0; j < 8; j++) y[j] = (f16)(acc_o[rt][c + j][e] * inv);
                    *(half8*)(o + c) = y;
                }
            } else {
                float* o = a.part_o + (u.slot_base + row) * D + 4 * r16;  // (part_dim's order)
#pragma unroll
                for (int c = 0; c < NT; c += 4)
                    *(float4v*)(o + 16 * c) = float4v{acc_o[rt][c][e], acc_o[rt][c + 1][e], acc_o[rt][c + 2][e], acc_o[rt][c + 3][e]};
            }
        }
    }
}

// Units of at most 16 rows: nothing to share through LDS, so each wave reads 32-key chunks of its
// own (chunk c of the unit's keys to wave c mod 8) straight into MFMA operands - K rows as A, a lane
// (g, r16) taking dims D/4 g .. of its key, V's 8-key blocks as B - and requests the next chunk's K
// once this one's scores are formed, its V once this one's P . V is; the waves' sums join through
// LDS. Bound by HBM latency and the dequantization between the loads: 6 rows over 32k 4-bit keys, D = 256,
// 38 MB in 14.4 us, 2.6 TB/s (a second chunk in flight does not fit the registers: 19.2 us with its
// spills). fp16: K's loads flat ones, at D = 256 19 spilled registers. Turbo4: K and V through the table of
// centroid pairs in LDS; the call with weights takes 23.6 us where the kernel for many rows and a second sight of
// K took 53.5, and 17.2 over 4-bit codes.
template <int KIND, int D, bool FAST, bool T4 = false>
__device__ __forceinline__ void few_body(const SharedArgs& a, char* lds) {
    constexpr int NM = D / 32, NT = D / 16, NG = D / kGroup, DG = D / 4, DPL = D / 16;
    constexpr int KP = DG * KIND / 128, VP = DPL * KIND / 16, E = 16 / KIND;  // 16-byte pieces a lane; dims a piece of V
    const Unit u = this_unit<D>(a);
    const int rows = u.row_end - u.row0, cap = u.cap, lo = u.lo, hc = u.hc, h = u.h, row_base = u.row0;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    const uint32_t magic = vconst(kMagic);
    constexpr int kSums = (16 * kWaves * 2 + kWaves * 16 * D) * 4;  // the waves' sums, joined at the end
    float2* const cp = (float2*)(lds + kSums);  // T4: a byte's two centroids
    static_assert(kSums + 256 * sizeof(float2) <= kSharedLds, "the waves' sums and the centroid pairs fit");
    if constexpr (T4) {
        const float* const cb = (int)blockIdx.x >= a.seg[0].n_units ? a.seg[1].t4_cb : a.seg[0].t4_cb;
        if (tid < 256) cp[tid] = float2{cb[tid & 15], cb[tid >> 4]};
        __syncthreads();
    }
    const bool row_ok = r16 < rows;
    const int rr = row_ok ? r16 : 0, lim = row_ok ? u.limit(row_base + rr, a.G) : -1, first_lim = u.limit(row_base, a.G);
    const int k_begin = max(u.k_begin, lo / 32 * 32), k_end = u.k_end;
    half8 qb[NM];
#pragma unroll
    for (int m = 0; m < NM; m++) {
        const u32x4 w = *(const u32x4*)(a.q + q_row(a, h, row_base + rr) * D + 8 * k_chunk<KIND>(m, g));
        qb[m] = as_h8(q_piece<T4 ? 16 : KIND>(row_ok ? w : u32x4{0, 0, 0, 0}, a.q_flip));
    }
    const uint32_t code_off = u.code_off;
    const int64_t krow0 = (int64_t)hc * cap + 8 * (r16 >> 2) + (r16 & 3), vblk0 = (int64_t)hc * (cap / 8) + g;
    const u32x4* const ksrc = (const u32x4*)(u.k_data + krow0 * (D * KIND / 32)) + g;
    const uint32_t* const kpsrc = KIND == 16 ? nullptr : u.k_params + krow0 * (T4 ? 1 : NG);
    const u32x4* const vsrc = (const u32x4*)(u.v_data + vblk0 * (D * KIND / 4)) + r16;
    const u32x4* const vpsrc =
        KIND == 16 ? nullptr : (const u32x4*)(u.v_params + (T4 ? vblk0 : vblk0 * NG + r16 * DPL / kGroup) * 8);
    // T4: V row-major, dims DPL n .. of the block's 8 rows
    const uint32_t* const vtsrc = T4 ? u.v_data + vblk0 * D + r16 * (DPL / 8) : nullptr;
    uint32_t vt[T4 ? 8 : 1][DPL / 8];
    u32x4 kc[2][KP], vc[VP], vp[2];
    uint32_t kp[2][KP];
    auto load_k = [&](int key) {
#pragma unroll
        for (int tt = 0; tt < 2; tt++)
#pragma unroll
            for (int i = 0; i < KP; i++) {
                kc[tt][i] = ksrc[(int64_t)(key + 4 * tt) * (D * KIND / 128) + 4 * i];
                if constexpr (T4)
                    kp[tt][i] = kpsrc[key + 4 * tt];
                else if constexpr (KIND != 16)
                    kp[tt][i] = kpsrc[(int64_t)(key + 4 * tt) * NG + k_param_slot(k_piece_group<KIND>(i, g), NG)];
            }
    };
    auto load_v = [&](int key) {
        if constexpr (T4) {
#pragma unroll
            for (int i = 0; i < 8; i++)
#pragma unroll
                for (int w = 0; w < DPL / 8; w++) vt[i][w] = vtsrc[(int64_t)(key + i) * (D / 8) + w];
            vp[0] = vpsrc[(int64_t)(key / 8) * 2];
            vp[1] = vpsrc[(int64_t)(key / 8) * 2 + 1];
            return;
        }
        // piece j holds slots 16 E j + E n ..: dims DPL n + E j .. of column n
#pragma unroll
        for (int j = 0; j < VP; j++) vc[j] = vsrc[(int64_t)(key / 8) * (D * KIND / 16) + 16 * j];
        if constexpr (KIND != 16) {
            vp[0] = vpsrc[(int64_t)(key / 8) * (NG * 2)];
            vp[1] = vpsrc[(int64_t)(key / 8) * (NG * 2) + 1];
        }
    };
    float m_run = -INFINITY, l_run = 0.0f;
    float4v acc_o[NT];
#pragma unroll
    for (int mm = 0; mm < NT; mm++) acc_o[mm] = float4v{0.f, 0.f, 0.f, 0.f};
    int key = k_begin + 32 * wave;
    if (key < k_end) {
        load_k(key);
        load_v(key);
    }
    for (; key < k_end; key += 32 * kWaves) {
        const bool more = key + 32 * kWaves < k_end;
        float4v acc[2] = {float4v{0.f, 0.f, 0.f, 0.f}, float4v{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int tt = 0; tt < 2; tt++) {
            PairConsts pc;
#pragma unroll
            for (int m = 0; m < NM; m++) {
                if constexpr (KIND != 16 && !T4)
                    if (m % E == 0) {
                        const half2v sb = h2(kp[tt][m / E]), s = {sb.x, sb.x}, b = {sb.y, sb.y};
                        pc = make_consts<FAST, KIND>(s, s, s, s, b, b, b, b, code_off);
                    }
                half8 ka;
                if constexpr (KIND == 16) {
                    ka = as_h8(kc[tt][m]);
                } else if constexpr (T4) {
                    const float kr = (float)h2(kp[tt][0]).x;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float2 c = cp[kc[tt][m / 4][m % 4] >> (8 * i) & 0xFFu];
                        ka[2 * i] = t4_f16_product(c.x, kr);
                        ka[2 * i + 1] = t4_f16_product(c.y, kr);
                    }
                } else if constexpr (KIND == 8)
                    ka = deq8<FAST>(kc[tt][m / 2][2 * m % 4], kc[tt][m / 2][2 * m % 4 + 1], pc);
                else
                    ka = deq4<FAST>(kc[tt][m / 4][m % 4], pc, magic);
                acc[tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qb[m], acc[tt], 0, 0, 0);
            }
        }
        if (more) load_k(key + 32 * kWaves);
        float s[8];
#pragma unroll
        for (int e = 0; e < 8; e++) s[e] = acc[e >> 2][e & 3] * a.scale2;
        if (a.scores && row_ok) {
            float4v* to = (float4v*)(a.scores + ((int64_t)h * a.R + row_base + r16) * a.score_stride + key + 8 * g);
            to[0] = float4v{s[0], s[1], s[2], s[3]};
            to[1] = float4v{s[4], s[5], s[6], s[7]};
        }
        const bool edge = key < lo || key + 31 > first_lim;
        if (edge) {
            asm volatile("");  // a branch, not selects in every step
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (key + 8 * g + e > lim || key + 8 * g + e < lo) s[e] = -INFINITY;
        }
        float mx = s[0];
#pragma unroll
        for (int e = 1; e < 8; e++) mx = fmaxf(mx, s[e]);
        if (__any(mx > m_run)) {
            const float m_new = fmaxf(m_run, wave_max_g(mx));
            const float alpha = m_run == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run - m_new);
            l_run *= alpha;
            float f[4];
#pragma unroll
            for (int e = 0; e < 4; e++) f[e] = __shfl(alpha, 4 * g + e);
#pragma unroll
            for (int mm = 0; mm < NT; mm++)
#pragma unroll
                for (int e = 0; e < 4; e++) acc_o[mm][e] *= f[e];
            m_run = m_new;
        }
        const float mref = m_run == -INFINITY ? 0.0f : m_run;
        half8 p16;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float p = __builtin_amdgcn_exp2f(s[e] - mref);
            l_run += p;
            p16[e] = (f16)p;
        }
        if constexpr (T4) {
            u32x4 keep = {~0u, ~0u, ~0u, ~0u};
            if (edge) keep = keep_keys(u.hi - (key + 8 * g)) & ~keep_keys(lo - (key + 8 * g));
#pragma unroll
            for (int j = 0; j < NT / 2; j++) {  // two dims
                half8 y0, y1;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float vr = (float)h2(vp[i / 4][i % 4]).y;
                    const float2 c = cp[vt[i][j / 4] >> (8 * (j % 4)) & 0xFFu];
                    y0[i] = t4_f16_product(c.x, vr);
                    y1[i] = t4_f16_product(c.y, vr);
                }
                y0 = as_h8(__builtin_bit_cast(u32x4, y0) & keep);  // hidden keys: 0 x inf is NaN
                y1 = as_h8(__builtin_bit_cast(u32x4, y1) & keep);
                acc_o[2 * j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(p16, y0, acc_o[2 * j], 0, 0, 0);
                acc_o[2 * j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(p16, y1, acc_o[2 * j + 1], 0, 0, 0);
            }
            if (more) load_v(key + 32 * kWaves);
            continue;
        }
        PairConsts pc;
        if constexpr (KIND != 16)
            pc = make_consts<FAST, KIND>(h2(vp[0][0]), h2(vp[0][1]), h2(vp[0][2]), h2(vp[0][3]), h2(vp[1][0]), h2(vp[1][1]),
                                         h2(vp[1][2]), h2(vp[1][3]), code_off);
#pragma unroll
        for (int j = 0; j < VP; j++) {
            half8 y[E];
#pragma unroll
            for (int i = 0; i < E; i++)
                y[i] = KIND == 16  ? as_h8(vc[j])
                       : KIND == 8 ? deq8<FAST>(vc[j][2 * i % 4], vc[j][(2 * i + 1) % 4], pc)
                                   : deq4<FAST>(vc[j][i % 4], pc, magic);
            if (edge) {  // hidden keys have weight 0, but 0 x inf is NaN
                asm volatile("");
                const u32x4 keep = keep_keys(u.hi - (key + 8 * g)) & ~keep_keys(lo - (key + 8 * g));
#pragma unroll
                for (int i = 0; i < E; i++) y[i] = as_h8(__builtin_bit_cast(u32x4, y[i]) & keep);
            }
#pragma unroll
            for (int i = 0; i < E; i++)
                acc_o[E * j + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(p16, y[i], acc_o[E * j + i], 0, 0, 0);
        }
        if (more) load_v(key + 32 * kWaves);
    }
    // the waves' sums against one maximum: m of all waves, then O and l rescaled, parked, added up
    float* const s_m = (float*)lds;                    // [8 waves][16 rows]
    float* const s_l = s_m + 16 * kWaves;              // [8][16]
    float* const s_o = s_l + 16 * kWaves;              // [8][rows][D]
    if (g == 0) s_m[16 * wave + r16] = m_run;
    __syncthreads();
    float M = -INFINITY;
#pragma unroll
    for (int v = 0; v < kWaves; v++) M = fmaxf(M, s_m[16 * v + r16]);
    const float f = __builtin_amdgcn_exp2f(m_run - (M == -INFINITY ? 0.0f : M));
    const float l = wave_sum_g(l_run) * f;
    if (g == 0) s_l[16 * wave + r16] = l;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float fe = __shfl(f, 4 * g + e);
        if (4 * g + e >= rows) continue;
        float* o = s_o + (wave * rows + 4 * g + e) * D + 4 * r16;  // (part_dim's order)
#pragma unroll
        for (int c = 0; c < NT; c += 4)
            *(float4v*)(o + 16 * c) = float4v{acc_o[c][e] * fe, acc_o[c + 1][e] * fe, acc_o[c + 2][e] * fe, acc_o[c + 3][e] * fe};
    }
    __syncthreads();
    const int64_t pbase = u.slot_base + row_base;
    for (int i = tid; i < rows * (D / 4); i += 64 * kWaves) {
        const int row = i / (D / 4), c = i % (D / 4);
        float4v o = {0.f, 0.f, 0.f, 0.f};
        float lr = 0.0f, mr = -INFINITY;
#pragma unroll
        for (int v = 0; v < kWaves; v++) {
            const float4v x = *(const float4v*)(s_o + (v * rows + row) * D + 4 * c);
#pragma unroll
            for (int j = 0; j < 4; j++) o[j] += x[j];
            lr += s_l[16 * v + row];
            mr = fmaxf(mr, s_m[16 * v + row]);
        }
        if (c == 0) a.part_ml[pbase + row] = float2{mr, lr};
        if (a.n_slots == 1) {
            const float inv = lr == 0.0f ? 0.0f : 1.0f / lr;
            half4v y;
#pragma unroll
            for (int j = 0; j < 4; j++) y[j] = (f16)(o[j] * inv);
            *(half4v*)(a.out + q_row(a, h, row_base + row) * D + part_dim<D>(c)) = y;
        } else {
            *(float4v*)(a.part_o + (pbase + row) * D + 4 * c) = o;
        }
    }
}

__device__ __forceinline__ bool unit_fast(const SharedArgs& a) {
    return *((int)blockIdx.x >= a.seg[0].n_units ? a.seg[1].fast_flag : a.seg[0].fast_flag) != 0;
}
template <int KIND, int D>
__global__ __launch_bounds__(64 * (kWaves + kFillWaves), 1) void shared_many_kernel(SharedArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    if constexpr (KIND != 16)
        if (unit_fast(a)) return many_body<KIND, D, true, false>(a, lds);
    many_body<KIND, D, false, false>(a, lds);
}
template <int D>
__global__ __launch_bounds__(64 * (kWaves + kFillWaves), 1) void shared_t4_many_kernel(SharedArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    many_body<4, D, false, false, true>(a, lds);
}
template <int D>
__global__ __launch_bounds__(64 * (kWaves + kFillWaves), 1) void shared_image_many_kernel(SharedArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    many_body<16, D, false, true>(a, lds);
}
// The key tiles of a cache as the kernel above copies them: grid (tiles, heads).
template <int KIND, int D>
__global__ __launch_bounds__(64 * kFillWaves) void shared_image_kernel(SharedSegment c, char* images) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    using S = BlockShape<D>;
    const int tid = threadIdx.x, t = blockIdx.x, hc = blockIdx.y;
    auto fill = [&](auto fast_c) {
        using Filler = TileFiller<KIND, D, decltype(fast_c)::value, true>;
        const Filler f(c, hc, t * S::KT, tid);
        typename Filler::Stage st;
        f.load(st, 0);
        f.store(st, lds, t * S::KT, 0, c.T);
    };
    if (*c.fast_flag)
        fill(std::true_type{});
    else
        fill(std::false_type{});
    __syncthreads();
    char* const to = images + ((int64_t)hc * c.n_tiles + t) * S::BUF;
    for (int i = 16 * tid; i < S::BUF; i += 16 * 64 * kFillWaves) *(u32x4*)(to + i) = *(const u32x4*)(lds + i);
}
template <int KIND, int D>
__global__ __launch_bounds__(64 * kWaves, 1) void shared_few_kernel(SharedArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    if constexpr (KIND != 16)
        if (unit_fast(a)) return few_body<KIND, D, true>(a, lds);
    few_body<KIND, D, false>(a, lds);
}
template <int D>
__global__ __launch_bounds__(64 * kWaves, 1) void shared_t4_few_kernel(SharedArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    few_body<4, D, false, true>(a, lds);
}

template <int D>
__global__ __launch_bounds__(256) void shared_merge_kernel(SharedArgs a) {
    __shared__ SharedMerge sm;
    merge_group<D>(a, blockIdx.x, blockIdx.y, sm);
}

// What a launch of n_pre units of a us and, behind them, n_tail units of b us takes on 256 CUs.
double makespan(int64_t n_pre, double a, int64_t n_tail, double b) {
    const int64_t full = n_pre / 256, rest = n_pre % 256;
    const double base = full * a;
    for (int k = 0;; k++) {  // the shortest time base + (rest ? a : 0) + k b that holds every tail unit
        const double t = base + (rest ? a : 0.0) + k * b;
        const int64_t fit = (256 - rest) * (int64_t)((t - base) / b + 1e-9) + rest * (int64_t)k;
        if (fit >= n_tail) return t;
        if (k > 64) return t + (double)(n_tail - fit) / 256 * b;
    }
}

void fill_cache(SharedSegment& s, const KVCache& c) {
    s.k_data = (const uint32_t*)c.k_data;
    s.k_params = c.k_params;
    s.v_data = (const uint32_t*)c.v_data;
    s.v_params = c.v_params;
    s.bits = c.bits;
    s.cap = c.cap;
    s.T = c.offset;
    s.code_off2 = c.code_offset2();
    s.fast_flag = c.fast_flag;
    s.t4_cb = c.turbo4() ? c.t4_tables + 4 * c.D : nullptr;
}

template <int KIND, int D>
int launch_images(const SharedArgs& a, hipStream_t stream) {
    const SharedSegment& c = a.seg[1];
    if (int rc = ensure_dynamic_lds((const void*)shared_image_kernel<KIND, D>, BlockShape<D>::BUF)) return rc;
    hipLaunchKernelGGL((shared_image_kernel<KIND, D>), dim3(c.n_tiles, c.heads), dim3(64 * kFillWaves),
                       BlockShape<D>::BUF, stream, c, (char*)c.images);
    QW_HIP_CHECK(hipGetLastError());
    if (int rc = ensure_dynamic_lds((const void*)shared_image_many_kernel<D>, kSharedLds)) return rc;
    hipLaunchKernelGGL((shared_image_many_kernel<D>), dim3(c.n_units), dim3(64 * (kWaves + kFillWaves)), kSharedLds,
                       stream, a);
    QW_HIP_CHECK(hipGetLastError());
    return QW_OK;
}
bool few_rows(const SharedArgs& a) {
    return std::max(a.seg[0].n_units ? a.seg[0].unit_rows : 0, a.seg[1].n_units ? a.seg[1].unit_rows : 0) <= kFewRows;
}
template <int KIND, int D>
int launch_units(const SharedArgs& a, hipStream_t stream) {
    if constexpr (KIND != 16)
        if (a.seg[1].images) return launch_images<KIND, D>(a, stream);
    const dim3 grid(a.seg[0].n_units + a.seg[1].n_units);
    const bool few = few_rows(a);
    const void* const kernel = few ? (const void*)shared_few_kernel<KIND, D> : (const void*)shared_many_kernel<KIND, D>;
    if (int rc = ensure_dynamic_lds(kernel, kSharedLds)) return rc;
    if (few)
        hipLaunchKernelGGL((shared_few_kernel<KIND, D>), grid, dim3(64 * kWaves), kSharedLds, stream, a);
    else
        hipLaunchKernelGGL((shared_many_kernel<KIND, D>), grid, dim3(64 * (kWaves + kFillWaves)), kSharedLds, stream, a);
    QW_HIP_CHECK(hipGetLastError());
    return QW_OK;
}

template <int D>
int launch_t4_units(const SharedArgs& a, hipStream_t stream) {
    const dim3 grid(a.seg[0].n_units + a.seg[1].n_units);
    const bool few = few_rows(a);
    const void* const kernel = few ? (const void*)shared_t4_few_kernel<D> : (const void*)shared_t4_many_kernel<D>;
    if (int rc = ensure_dynamic_lds(kernel, kSharedLds)) return rc;
    if (few)
        hipLaunchKernelGGL(shared_t4_few_kernel<D>, grid, dim3(64 * kWaves), kSharedLds, stream, a);
    else
        hipLaunchKernelGGL(shared_t4_many_kernel<D>, grid, dim3(64 * (kWaves + kFillWaves)), kSharedLds, stream, a);
    QW_HIP_CHECK(hipGetLastError());
    return QW_OK;
}
int launch_units(int bits, int D, const SharedArgs& a, hipStream_t stream) {
    if (a.seg[0].n_units + a.seg[1].n_units == 0) return QW_OK;
    if (a.seg[0].t4_cb || a.seg[1].t4_cb) return D == 256 ? launch_t4_units<256>(a, stream) : launch_t4_units<128>(a, stream);
    if (D == 256)
        return bits == 4   ? launch_units<4, 256>(a, stream)
               : bits == 8 ? launch_units<8, 256>(a, stream)
                           : launch_units<16, 256>(a, stream);
    return bits == 4   ? launch_units<4, 128>(a, stream)
           : bits == 8 ? launch_units<8, 128>(a, stream)
                       : launch_units<16, 128>(a, stream);
}

}  // namespace

int make_room(KVCache& c, int n_rows, hipStream_t stream) {
    const int64_t need = (int64_t)c.offset + n_rows;
    if (need <= c.cap) return QW_OK;
    QW_REQUIRE(need <= INT32_MAX - 256, QW_ERR_INVALID_ARGUMENT, "append: too many rows");
    hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
    QW_HIP_CHECK(hipStreamIsCapturing(stream, &cs));
    QW_REQUIRE(cs == hipStreamCaptureStatusNone, QW_ERR_STATE,
               "append: the cache has to grow and the stream is being captured; reserve it before");
    // (geometric, as KVCache::update grows it)
    return c.reserve((int)std::min<int64_t>(std::max(need, (int64_t)c.cap + c.cap / 2), INT32_MAX - 256), stream);
}

int plan_shared(const KVCache* prefix, const KVCache* tails, int tail_rows, const void* q, int n_seq, int n_rows, int G,
                int hkv, const int32_t* starts, float scale, bool causal, void* out, hipStream_t stream, SharedArgs* pa) {
    SharedArgs& a = *pa;
    a = SharedArgs{};
    const KVCache* c[2] = {prefix && prefix->offset > 0 ? prefix : nullptr, tails && tail_rows > 0 ? tails : nullptr};
    const int D = (prefix ? prefix : tails)->D, KT = shared_tile(D);
    a.q = (const f16*)q;
    a.out = (f16*)out;
    a.starts = starts;
    a.Tq = n_rows;
    a.G = G;
    a.hkv = hkv;
    // (a merge of a workgroup of 256 a row stays below 2^32 threads)
    // (n_seq * n_rows is below 2^62; times G it could pass 2^63)
    const int64_t seq_rows = (int64_t)n_seq * n_rows;
    QW_REQUIRE(seq_rows < 1 << 24 && seq_rows * G < 1 << 24, QW_ERR_UNSUPPORTED,
               "attention: 2^24 or more rows a KV head in one call");
    a.R = n_seq * n_rows * G;
    // (over Turbo4 caches q and the output pass through launches of a wave a row)
    QW_REQUIRE(!(prefix ? prefix : tails)->turbo4() || (int64_t)a.R * hkv <= UINT32_MAX / 64 - 3, QW_ERR_UNSUPPORTED,
               "attention over a Turbo4 cache: about 2^26 or more query rows in one call");
    // (a scale of 0 stands as a tiny one, which leaves every score 0 and a hidden key's -inf itself; one that
    // passes fp32 times log2 e as its largest number, which leaves a score of 0 itself)
    a.scale2 = std::min(std::max(std::fabs(scale) * kLog2e, 1e-37f), FLT_MAX);
    a.q_flip = scale < 0.0f ? 0x80008000u : 0u;
    int tiles[2] = {0, 0}, n_qt[2] = {0, 0};
    for (int i = 0; i < 2; i++) {
        SharedSegment& s = a.seg[i];
        s.n_split = s.heads = 1;
        if (!c[i]) continue;
        fill_cache(s, *c[i]);
        if (i == 1) s.T = tail_rows;
        s.heads = c[i]->hkv;
        s.rows = i == 0 ? a.R : n_rows * G;
        // query tiles of equal size, in row tiles (few rows: one)
        const int wave_rows = 16 * many_tiles(D), rt = (s.rows + wave_rows - 1) / wave_rows;
        n_qt[i] = (rt + kWaves - 1) / kWaves;
        s.unit_rows = s.rows <= kFewRows ? s.rows : wave_rows * ((rt + n_qt[i] - 1) / n_qt[i]);
        s.causal_rows = i == 1 && causal ? n_rows : 0;
        tiles[i] = (s.T + KT - 1) / KT;
    }
    // One quantized cache under many query tiles: its key tiles are dequantized once, into images
    // (1.03 times its fp16 K and V: 2.2 GB at most), not once a query tile.
    const bool images = c[1] && !c[0] && !starts && c[1]->affine() && n_qt[1] >= kImageQueryTiles &&
                        (int64_t)c[1]->hkv * tail_rows * D <= (int64_t)1 << 29;
    // Tiles a split, for each launch: the count with the shortest estimate. A unit's us: a start and an
    // end that grow with its rows, and a time a tile (measured: 30 and 126 rows of 8-bit keys at D = 256
    // 23.6 and 38.4 us in 8 tiles, 126 rows 103 us in 32; few rows 14.5 us in 9); a partial row costs its
    // write and its read by the merge.
    a.n_slots = 0;
    auto plan = [&](std::initializer_list<int> in) -> int {
        bool few = true;
        int most = 0;
        for (int i : in)
            if (c[i]) {
                few = few && a.seg[i].unit_rows <= kFewRows;
                most = std::max(most, tiles[i]);
            }
        auto unit_us = [&](int i, int n) {
            const SharedSegment& s = a.seg[i];
            if (few) return 5.0 + 0.65 * n;
            const double fill = (double)s.unit_rows / (16 * many_tiles(D) * kWaves);
            return 6.0 + 4.0 * fill + n * (images ? 1.9 : 1.0 + 1.5 * fill + (s.bits == 16 ? 0.6 : 0.0));
        };
        int best = most;
        double best_cost = 1e30;
        for (int tps = 1; tps <= most; tps += std::max(1, tps / 16)) {
            double us[2] = {0.0, 1.0};
            int64_t units[2] = {0, 0};
            int slots = 0;
            for (int i : in) {
                if (!c[i]) continue;
                const int n = (tiles[i] + tps - 1) / tps;
                us[i] = unit_us(i, std::min(tps, tiles[i]));
                units[i] = (int64_t)n_qt[i] * a.seg[i].heads * n;
                slots += n;
            }
            if (slots > kSharedMaxSlots) continue;
            const double cost = makespan(units[0], us[0], units[1], us[1]) + 1.8e-6 * slots * a.R * hkv * D;
            if (cost < best_cost) {
                best_cost = cost;
                best = tps;
            }
        }
        for (int i : in) {
            SharedSegment& s = a.seg[i];
            if (!c[i]) continue;
            s.tiles_per_split = best;
            s.n_split = (tiles[i] + best - 1) / best;
            s.slot0 = a.n_slots;
            a.n_slots += s.n_split;
            const int64_t units = (int64_t)n_qt[i] * s.heads * s.n_split;
            // (both caches' units in one launch of fewer than 2^32 threads)
            QW_REQUIRE(units <= UINT32_MAX / (64 * (kWaves + kFillWaves)) / 2, QW_ERR_UNSUPPORTED,
                       "shared attention: too many rows for one call");
            s.n_units = (int)units;
        }
        return QW_OK;
    };
    if (c[0] && c[1] && c[0]->bits != c[1]->bits) {
        if (int rc = plan({0})) return rc;
        if (int rc = plan({1})) return rc;
    } else if (int rc = plan({0, 1})) {
        return rc;
    }
    const size_t rows = (size_t)a.n_slots * hkv * a.R;
    const size_t o_bytes = a.n_slots > 1 ? rows * D * sizeof(float) : 0, ml_bytes = (rows * sizeof(float2) + 15) / 16 * 16;
    const size_t img_bytes = images ? (size_t)a.seg[1].heads * tiles[1] * (D == 256 ? BlockShape<256>::BUF : BlockShape<128>::BUF) : 0;
    void* ws = nullptr;
    if (int rc = workspace(kWsShared, (prefix ? prefix : tails)->device, stream, o_bytes + ml_bytes + img_bytes, &ws))
        return rc;
    a.part_o = (float*)ws;
    a.part_ml = (float2*)((char*)ws + o_bytes);
    if (images) a.seg[1].images = (const char*)ws + o_bytes + ml_bytes;
    a.seg[1].n_tiles = tiles[1];
    return QW_OK;
}

int launch_shared(const KVCache* prefix, const KVCache* tails, const SharedArgs& a, hipStream_t stream) {
    const int D = (prefix ? prefix : tails)->D;
    const int b0 = a.seg[0].n_units ? prefix->bits : 0, b1 = a.seg[1].n_units ? tails->bits : 0;
    if (b0 == b1 || !b0 || !b1) return launch_units(std::max(b0, b1), D, a, stream);
    // caches of different widths: a launch each
    SharedArgs x = a;
    x.seg[1].n_units = 0;
    if (int rc = launch_units(b0, D, x, stream)) return rc;
    x.seg[1].n_units = a.seg[1].n_units;
    x.seg[0].n_units = 0;
    return launch_units(b1, D, x, stream);
}

int launch_shared_merge(int D, const SharedArgs& a, hipStream_t stream) {
    if (a.n_slots == 1) return QW_OK;
    const dim3 grid(merge_groups(D, a.R, a.hkv, a.n_slots), a.hkv);
    if (D == 256)
        hipLaunchKernelGGL(shared_merge_kernel<256>, grid, dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL(shared_merge_kernel<128>, grid, dim3(256), 0, stream, a);
    QW_HIP_CHECK(hipGetLastError());
    return QW_OK;
}

int shared_turbo4_room(const KVCache& c, int64_t q_rows, hipStream_t stream, SharedArgs* a) {
    void* ws = nullptr;
    if (int rc = workspace(kWsTurbo4, c.device, stream, 2 * (size_t)q_rows * c.D * sizeof(f16), &ws)) return rc;
    a->q = (const f16*)ws;
    a->out = (f16*)ws + q_rows * c.D;
    return QW_OK;
}
int shared_turbo4_rotate_q(const KVCache& c, const void* q, int64_t q_rows, const SharedArgs& a, hipStream_t stream) {
    return launch_turbo4_rotate(c, (const f16*)q, (int)q_rows, false, (f16*)a.q, stream);
}

static int check_shared(const KVCache& p, const KVCache* t, int n_seq, const void* q, int n_q_heads, int n_rows,
                        float scale, const void* out, int64_t tail_rows) {
    QW_REQUIRE(q && out, QW_ERR_INVALID_ARGUMENT, "shared attention: null q/out");
    QW_REQUIRE(n_seq > 0 && n_rows > 0 && n_q_heads > 0 && n_q_heads % p.hkv == 0, QW_ERR_INVALID_ARGUMENT,
               "shared attention: n_seq, n_rows > 0 and n_q_heads a positive multiple of n_kv_heads");
    const int64_t seq_rows = (int64_t)n_seq * n_rows;
    QW_REQUIRE(seq_rows <= INT32_MAX / 2 && seq_rows * (n_q_heads / p.hkv) <= INT32_MAX / 2, QW_ERR_INVALID_ARGUMENT,
               "shared attention: too many rows");
    QW_REQUIRE(std::isfinite(scale), QW_ERR_INVALID_ARGUMENT, "shared attention: scale must be finite");
    if (t) {
        QW_REQUIRE(t != &p, QW_ERR_INVALID_ARGUMENT, "shared attention: the prefix and the tails are one cache");
        QW_REQUIRE((int64_t)n_seq * p.hkv == t->hkv && t->D == p.D && t->device == p.device, QW_ERR_INVALID_ARGUMENT,
                   "shared attention: the tails need n_seq * n_kv_heads heads of the prefix's head_dim, on its device");
        QW_REQUIRE(t->turbo4() == p.turbo4() && (!p.turbo4() || t->turbo_seed == p.turbo_seed), QW_ERR_UNSUPPORTED,
                   "shared attention: Turbo4 caches go with Turbo4 caches of their seed");
        QW_REQUIRE(tail_rows == 0 || tail_rows >= n_rows, QW_ERR_INVALID_ARGUMENT,
                   "shared attention: fewer tail rows than query rows");
    }
    QW_REQUIRE(p.offset > 0 || tail_rows > 0, QW_ERR_INVALID_ARGUMENT, "shared attention: no cached rows");
    return QW_OK;
}

int shared_attention(KVCache& prefix, KVCache* tails, int n_seq, const int32_t* starts, const void* q, int n_q_heads,
                     int n_rows, const void* k_new, const void* v_new, float scale, void* out, hipStream_t stream) {
    const bool append = k_new || v_new;
    QW_REQUIRE(!append || (tails && k_new && v_new), QW_ERR_INVALID_ARGUMENT,
               "shared attention: an append needs tails, k_new and v_new");
    const int64_t tail_rows = tails ? (int64_t)tails->offset + (append ? n_rows : 0) : 0;
    if (int rc = check_shared(prefix, tails, n_seq, q, n_q_heads, n_rows, scale, out, tail_rows)) return rc;
    DeviceGuard dg(prefix.device);
    QW_REQUIRE(dg.ok, QW_ERR_HIP, "shared attention: hipSetDevice failed");
    // (what can fail for want of memory comes before the append)
    if (append)
        if (int rc = make_room(*tails, n_rows, stream)) return rc;
    SharedArgs a;
    if (int rc = plan_shared(&prefix, tails, (int)tail_rows, q, n_seq, n_rows, n_q_heads / prefix.hkv, prefix.hkv, starts, scale, true,
                             out, stream, &a))
        return rc;
    const int64_t q_rows = (int64_t)n_seq * n_q_heads * n_rows;
    if (prefix.turbo4())
        if (int rc = shared_turbo4_room(prefix, q_rows, stream, &a)) return rc;
    if (append)
        if (int rc = tails->update(k_new, v_new, n_rows, stream)) return rc;
    if (prefix.turbo4())
        if (int rc = shared_turbo4_rotate_q(prefix, q, q_rows, a, stream)) return rc;
    if (int rc = launch_shared(&prefix, tails, a, stream)) return rc;
    if (int rc = launch_shared_merge(prefix.D, a, stream)) return rc;
    return prefix.turbo4() ? launch_turbo4_rotate(prefix, a.out, (int)q_rows, true, (f16*)out, stream) : QW_OK;
}

}  // namespace qw
