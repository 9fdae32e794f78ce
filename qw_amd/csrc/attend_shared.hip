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
// tails, each seen by Tq G rows, are units of one launch, both cut into key
// splits, and a second launch joins the partials.
//
// A unit (a workgroup of 8 waves): up to 128 rows of one head over a run of key
// tiles (KT = 16384 / D keys, the LDS layout of block_tile.hpp). In round i the
// workgroup dequantizes tile i + 1 (its codes in registers) into the free one of
// two LDS buffers, requests the codes of a later tile and computes tile i:
//   S^T = K . Q^T (v_mfma_f32_16x16x32_f16; a lane then holds 8 consecutive keys
//   of one row, the A operand of P . V), scores scaled and kept in fp32, online
//   softmax against the running maximum (the largest weight is exactly 1), P
//   rounded to fp16 for O += P . V, O in fp32.
// Rounded to fewer than 32 bits: P, to fp16 (2^-12 relative rms a weight, and
// averaged over the keys; the output's own rounding is the larger), and the
// output. Workgroups of fewer than 8 row tiles give the free waves halves or
// quarters of each tile's keys and join them through LDS.
#include <algorithm>
#include <cmath>

#include "attend_shared.hpp"
#include "block_tile.hpp"
#include "dequant.hpp"
#include "kv_cache.hpp"

namespace qw {

namespace {

constexpr int kWaves = 8, kFewRows = 16;

// KIND: 16, 8 (affine and Int8) or 4 bits.
template <int KIND, int D, bool FAST>
__device__ __forceinline__ void shared_body(const SharedArgs& a, char* lds) {
    using S = BlockShape<D>;
    constexpr int KT = S::KT, NSUB = S::NSUB, NM = S::NM, NT = S::NT, NG = S::NG;
    constexpr int TPR = S::TPR, LTPR = S::LTPR, TPB = S::TPB, BUF = S::BUF, KBUF = S::KBUF, VROW = S::VROW;
    constexpr int KU = KIND / 4;               // 16-byte loads of a 32-dim K slice / 4-slot V slice
    constexpr int NST = 2;                     // register stages: tiles of codes in flight
    static_assert(KT * TPR == 64 * kWaves && (KT / 8) * TPB == 64 * kWaves, "a slice of each kind a thread");
    // ---- the unit: a split of a query tile of a head of one of the two caches
    const bool is_tail = (int)blockIdx.x >= a.seg[0].n_units;
    const int u_id = (int)blockIdx.x - (is_tail ? a.seg[0].n_units : 0);
#define QW_SEG(f) (is_tail ? a.seg[1].f : a.seg[0].f)
    const int n_split = QW_SEG(n_split), heads = QW_SEG(heads), T = QW_SEG(T), cap = QW_SEG(cap);
    const int sp = u_id % n_split, hc = u_id / n_split % heads, qt = u_id / n_split / heads;
    const int h = hc % a.hkv, seg_rows = QW_SEG(rows), unit_rows = QW_SEG(unit_rows);
    const int row_base = hc / a.hkv * seg_rows;  // the head's rows of its KV head's R
    const int row0 = row_base + qt * unit_rows;
    const int row_end = row_base + min(seg_rows, (qt + 1) * unit_rows);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    const uint32_t magic = vconst(kMagic);

    // visible keys: [lo, hi) of the unit's rows together
    const int causal_rows = QW_SEG(causal_rows);  // 0: every key to T - 1
    int lo = 0;
    if (is_tail && a.starts) lo = min(max(a.starts[hc / a.hkv], 0), T);
    auto limit = [&](int row) {  // a row's last visible key
        return causal_rows ? T - causal_rows + (row - row_base) / a.G : T - 1;
    };
    const int hi = limit(row_end - 1) + 1;
    const int tps = QW_SEG(tiles_per_split);
    const int t0 = lo / KT + sp * tps, t1 = min((hi + KT - 1) / KT, t0 + tps);
    const int n = max(t1 - t0, 0);

    // ---- waves: row tile and part of each tile's keys
    const int n_rt = (row_end - row0 + 15) / 16;
    const int lrt = n_rt <= 1 ? 0 : n_rt <= 2 ? 1 : n_rt <= 4 ? 2 : 3;  // log2 of the row tiles, padded
    const int parts = min(kWaves >> lrt, NSUB);
    const int part = wave >> lrt, wrow0 = row0 + 16 * (wave & ((1 << lrt) - 1));
    const bool live = part < parts && wrow0 < row_end;
    const int rho = wrow0 + r16;
    const bool row_ok = live && rho < row_end;
    const int lim = row_ok ? limit(rho) : -1;
    const int wave_first_lim = limit(min(wrow0, row_end - 1)), wave_lim = limit(min(wrow0 + 15, row_end - 1));

    half8 qb[NM];
    {
        const int row = row_ok ? rho : row0, seq = row / (a.Tq * a.G), rr = row % (a.Tq * a.G);
        const f16* qrow = a.q + (((int64_t)seq * a.hkv * a.G + h * a.G + rr % a.G) * a.Tq + rr / a.G) * D;
#pragma unroll
        for (int m = 0; m < NM; m++) {
            u32x4 w = *(const u32x4*)(qrow + 32 * m + 8 * g);
            if (!row_ok) w = u32x4{0, 0, 0, 0};
            if constexpr (KIND == 4)  // K rows sit in LDS as dim pairs (0,4),(1,5),(2,6),(3,7)
                w = u32x4{__builtin_amdgcn_perm(w.z, w.x, 0x05040100u), __builtin_amdgcn_perm(w.z, w.x, 0x07060302u),
                          __builtin_amdgcn_perm(w.w, w.y, 0x05040100u), __builtin_amdgcn_perm(w.w, w.y, 0x07060302u)};
            qb[m] = as_h8(w);
        }
    }

    // ---- tile loads: key kk's 32-dim slice q32, V block vb's 4 physical slots from 4 vj
    struct Stage {
        u32x4 kc[KU], vc[KU], vp[2];
        uint32_t kp;
    };
    const int q32 = (tid >> 4) & (TPR - 1), kk = (tid & 15) | ((tid >> (4 + LTPR)) << 4);
    const int vb = tid / TPB, vj = tid % TPB;
    // slots 4 vj .. + 3 are dims vd + step e (KIND 8: two dims of two lane groups)
    constexpr int DPL = D / 16;
    const int vn = KIND == 16 ? 0 : KIND == 8 ? (2 * vj) % 16 : vj % 16;
    const int vr = KIND == 8 ? 2 * (vj / 8) : 4 * (vj / 16);
    const int64_t krow = (int64_t)hc * cap + kk, vblk = (int64_t)hc * (cap / 8) + vb;
    const u32x4* const ksrc = (const u32x4*)(QW_SEG(k_data) + krow * (D * KIND / 32)) + KU * q32;
    const u32x4* const vsrc = (const u32x4*)(QW_SEG(v_data) + vblk * (D * KIND / 4)) + KU * vj;
    const uint32_t* const kpsrc = KIND == 16 ? nullptr : QW_SEG(k_params) + krow * NG + k_param_slot(q32 >> 1, NG);
    const u32x4* const vpsrc =
        KIND == 16 ? nullptr : (const u32x4*)(QW_SEG(v_params) + (vblk * NG + vn * DPL / kGroup) * 8);
    auto load = [&](Stage& st, int i) {
        const int64_t rows = (int64_t)(t0 + i) * KT, blks = rows / 8;
#pragma unroll
        for (int u = 0; u < KU; u++) st.kc[u] = ksrc[rows * (D * KIND / 128) + u];
#pragma unroll
        for (int u = 0; u < KU; u++) st.vc[u] = vsrc[blks * (D * KIND / 16) + u];
        if constexpr (KIND != 16) {
            st.kp = kpsrc[rows * NG];
            st.vp[0] = vpsrc[blks * (NG * 2)];
            st.vp[1] = vpsrc[blks * (NG * 2) + 1];
        }
    };
    const uint32_t code_off = QW_SEG(code_off2);
    // Tile i dequantized into buffer i & 1: f16(f16(code * scale) + bias), as the fetch gives
    // it; V in the fp16 slot order whatever the codes'. Keys outside [lo, hi) go in as
    // zeros of V: they have weight 0, but 0 x inf is NaN.
    auto store = [&](const Stage& st, int i) {
        half8* const sK = (half8*)(lds + BUF * (i & 1));
        half8* const sV = (half8*)(lds + BUF * (i & 1) + KBUF) + vb * VROW;
        half8* const kdst = sK + kaddr<KT>(kk, 4 * q32);
        if constexpr (KIND == 16) {
#pragma unroll
            for (int w = 0; w < 4; w++) kdst[w * KT] = as_h8(st.kc[w]);
        } else {
            const half2v sb = h2(st.kp), s = {sb.x, sb.x}, b = {sb.y, sb.y};
            const PairConsts c = make_consts<FAST, KIND>(s, s, s, s, b, b, b, b, code_off);
#pragma unroll
            for (int w = 0; w < 4; w++)
                kdst[w * KT] = KIND == 4 ? deq4<FAST>(st.kc[0][w], c, magic)
                                         : deq8<FAST>(st.kc[KU / 2 * (w / 2)][2 * (w % 2)],
                                                       st.kc[KU / 2 * (w / 2)][2 * (w % 2) + 1], c);
        }
        half8 y[4];
        if constexpr (KIND == 16) {
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = as_h8(st.vc[e]);
        } else {
            const PairConsts c = make_consts<FAST, KIND>(h2(st.vp[0][0]), h2(st.vp[0][1]), h2(st.vp[0][2]), h2(st.vp[0][3]),
                                                          h2(st.vp[1][0]), h2(st.vp[1][1]), h2(st.vp[1][2]), h2(st.vp[1][3]),
                                                          code_off);
#pragma unroll
            for (int e = 0; e < 4; e++)
                y[e] = KIND == 4 ? deq4<FAST>(st.vc[0][e], c, magic)
                                 : deq8<FAST>(st.vc[KU / 2 * (e / 2)][2 * (e % 2)],
                                               st.vc[KU / 2 * (e / 2)][2 * (e % 2) + 1], c);
        }
        const int key0 = (t0 + i) * KT;
        if (key0 < lo || key0 + KT > hi) {
            const u32x4 keep = keep_keys(hi - (key0 + 8 * vb)) & ~keep_keys(lo - (key0 + 8 * vb));
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = as_h8(__builtin_bit_cast(u32x4, y[e]) & keep);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int at = KIND == 16  ? 4 * vj + e + (vj >> 2)
                           : KIND == 8 ? 17 * (vr + e % 2) + vn + e / 2
                                       : 17 * (vr + e) + vn;
            sV[at] = y[e];
        }
    };

    float m_run = -INFINITY, l_run = 0.0f;  // log2 units; l: this lane's share
    float4v acc_o[NT];
#pragma unroll
    for (int mm = 0; mm < NT; mm++) acc_o[mm] = float4v{0.f, 0.f, 0.f, 0.f};

    // NU sub-blocks of 32 keys, from sub-block ub of tile i
    auto step = [&](int i, int ub, auto nu_c) {
        constexpr int NU = decltype(nu_c)::value;
        const half8* const sK = (const half8*)(lds + BUF * (i & 1)) + 32 * ub;
        const half8* const sV = (const half8*)(lds + BUF * (i & 1) + KBUF) + 4 * ub * VROW;
        const int kt0 = (t0 + i) * KT + 32 * ub;
        const int key0 = 8 * (r16 >> 2) + (r16 & 3), b4 = (key0 >> 4) & 1;
        const half8* const k0 = sK + g * KT + key0 + 4 * b4;
        const half8* const k1 = sK + g * KT + key0 + 4 * (b4 ^ 1);
        float4v acc[NU][2];
#pragma unroll
        for (int u = 0; u < NU; u++) acc[u][0] = acc[u][1] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int m = 0; m < NM; m++)
#pragma unroll
            for (int u = 0; u < NU; u++) {
                acc[u][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0[4 * m * KT + 32 * u], qb[m], acc[u][0], 0, 0, 0);
                acc[u][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1[4 * m * KT + 32 * u], qb[m], acc[u][1], 0, 0, 0);
            }
        float s[NU][8];
#pragma unroll
        for (int u = 0; u < NU; u++)
#pragma unroll
            for (int e = 0; e < 8; e++) s[u][e] = acc[u][e >> 2][e & 3] * a.scale2;
        if (kt0 + 32 * NU - 1 > wave_first_lim || kt0 < lo) {
#pragma unroll
            for (int u = 0; u < NU; u++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int key = kt0 + 32 * u + 8 * g + e;
                    if (key > lim || key < lo) s[u][e] = -INFINITY;
                }
        }
        float mx = s[0][0];
#pragma unroll
        for (int u = 0; u < NU; u++)
#pragma unroll
            for (int e = 0; e < 8; e++) mx = fmaxf(mx, s[u][e]);
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
        half8 p16[NU];
#pragma unroll
        for (int u = 0; u < NU; u++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float p = __builtin_amdgcn_exp2f(s[u][e] - mref);
                l_run += p;
                p16[u][e] = (f16)p;
            }
#pragma unroll
        for (int u = 0; u < NU; u++)
#pragma unroll
            for (int mm = 0; mm < NT; mm++)
                acc_o[mm] = __builtin_amdgcn_mfma_f32_16x16x32_f16(p16[u], sV[(4 * u + g) * VROW + r16 + 17 * mm],
                                                                   acc_o[mm], 0, 0, 0);
    };

    // ---- rounds: stage x holds tile i where i mod NST == x. A loop of its own for the waves
    // that take one sub-block of a tile and for those that take PER = 2 or 4 of them, two at a
    // time (one loop for both spilled registers); the barriers pair up all the same.
    auto rounds = [&](auto per_c) {
        constexpr int PER = decltype(per_c)::value, NU = PER < 2 ? 1 : 2;
        const int ub0 = part * PER;
        auto compute = [&](int i) {
#pragma unroll
            for (int ub = 0; ub < PER; ub += NU)
                if (live && (t0 + i) * KT + 32 * (ub0 + ub) <= wave_lim)
                    step(i, ub0 + ub, std::integral_constant<int, NU>{});
        };
        Stage st[NST];
        if (n > 0) {
#pragma unroll
            for (int x = 0; x < NST; x++)
                if (x < n) load(st[x], x);
            store(st[0], 0);
            if (NST < n) load(st[0], NST);
        }
        __syncthreads();
        for (int i = 0; i < n; i += NST) {
#pragma unroll
            for (int x = 0; x < NST; x++) {
                if (i + x >= n) break;
                if (i + x + 1 < n) {
                    store(st[(x + 1) % NST], i + x + 1);
                    if (i + x + 1 + NST < n) load(st[(x + 1) % NST], i + x + 1 + NST);
                }
                compute(i + x);
                __syncthreads();
            }
        }
    };
    if (parts == NSUB)
        rounds(std::integral_constant<int, 1>{});
    else if (NSUB == 2 || parts == 2)
        rounds(std::integral_constant<int, 2>{});
    else
        rounds(std::integral_constant<int, NSUB>{});

    // ---- the parts of a row tile joined in its part 0, through LDS
    float l = wave_sum_g(l_run);
    if (parts > 1) {
        constexpr int REG = 64 * NT * 16 + 64 * 8;
        static_assert(6 * REG <= 2 * BUF && 4 * REG <= 2 * BUF, "the parked parts fit the tile buffers");
        if (live && part > 0) {
            char* reg = lds + (wave - (1 << lrt)) * REG;
#pragma unroll
            for (int mm = 0; mm < NT; mm++) ((float4v*)reg)[mm * 64 + lane] = acc_o[mm];
            ((float2*)(reg + 64 * NT * 16))[lane] = float2{m_run, l};
        }
        __syncthreads();
        if (live && part == 0) {
            for (int p = 1; p < parts; p++) {
                const char* reg = lds + (((p - 1) << lrt) + wave) * REG;
                const float2 ml = ((const float2*)(reg + 64 * NT * 16))[lane];
                const float M = fmaxf(m_run, ml.x), mr = M == -INFINITY ? 0.0f : M;
                const float fa = __builtin_amdgcn_exp2f(m_run - mr), fb = __builtin_amdgcn_exp2f(ml.x - mr);
                l = l * fa + ml.y * fb;
                m_run = M;
                float xa[4], xb[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    xa[e] = __shfl(fa, 4 * g + e);
                    xb[e] = __shfl(fb, 4 * g + e);
                }
#pragma unroll
                for (int mm = 0; mm < NT; mm++) {
                    const float4v o = ((const float4v*)reg)[mm * 64 + lane];
#pragma unroll
                    for (int e = 0; e < 4; e++) acc_o[mm][e] = acc_o[mm][e] * xa[e] + o[e] * xb[e];
                }
            }
        }
    }
    if (!live || part > 0) return;

    // ---- rows out: lane (g, r16) holds dims NT r16 .. + NT - 1 of rows 4g + e
    const int64_t pbase = ((int64_t)(QW_SEG(slot0) + sp) * a.hkv + h) * a.R;
    if (g == 0 && row_ok) a.part_ml[pbase + rho] = float2{m_run, l};
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const int row = wrow0 + 4 * g + e;
        const float le = __shfl(l, 4 * g + e);
        if (row >= row_end) continue;
        if (a.n_slots == 1) {
            const float inv = le == 0.0f ? 0.0f : 1.0f / le;
            const int seq = row / (a.Tq * a.G), rr = row % (a.Tq * a.G);
            f16* o = a.out + (((int64_t)seq * a.hkv * a.G + h * a.G + rr % a.G) * a.Tq + rr / a.G) * D + NT * r16;
#pragma unroll
            for (int c = 0; c < NT; c += 8) {
                half8 y;
#pragma unroll
                for (int j = 0; j < 8; j++) y[j] = (f16)(acc_o[c + j][e] * inv);
                *(half8*)(o + c) = y;
            }
        } else {
            float* o = a.part_o + (pbase + row) * D + NT * r16;
#pragma unroll
            for (int c = 0; c < NT; c += 4)
                *(float4v*)(o + c) = float4v{acc_o[c][e], acc_o[c + 1][e], acc_o[c + 2][e], acc_o[c + 3][e]};
        }
    }
}

// Units of at most 16 rows: nothing to share through LDS, so each wave reads 32-key chunks of its
// own (chunk c of the unit's keys to wave c mod 8) straight into MFMA operands - K rows as A, a lane
// (g, r16) taking dims D/4 g .. of its key, V's 8-key blocks as B - and requests the next chunk's K
// once this one's scores are formed, its V once this one's P . V is. Bound by HBM latency and
// bandwidth; the waves' sums join through LDS.
template <int KIND, int D, bool FAST>
__device__ __forceinline__ void few_body(const SharedArgs& a, char* lds) {
    constexpr int NM = D / 32, NT = D / 16, NG = D / kGroup, DG = D / 4, DPL = D / 16;
    constexpr int KP = DG * KIND / 128, VP = DPL * KIND / 16, E = 16 / KIND;  // 16-byte pieces a lane; dims a piece of V
    const bool is_tail = (int)blockIdx.x >= a.seg[0].n_units;
    const int u_id = (int)blockIdx.x - (is_tail ? a.seg[0].n_units : 0);
    const int n_split = QW_SEG(n_split), heads = QW_SEG(heads), T = QW_SEG(T), cap = QW_SEG(cap);
    const int sp = u_id % n_split, hc = u_id / n_split;
    const int h = hc % a.hkv, rows = QW_SEG(rows), row_base = hc / a.hkv * rows;
    (void)heads;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    const uint32_t magic = vconst(kMagic);
    const int causal_rows = QW_SEG(causal_rows);
    int lo = 0;
    if (is_tail && a.starts) lo = min(max(a.starts[hc / a.hkv], 0), T);
    const bool row_ok = r16 < rows;
    const int rr = row_ok ? r16 : 0, lim = !row_ok ? -1 : causal_rows ? T - causal_rows + rr / a.G : T - 1;
    const int first_lim = causal_rows ? T - causal_rows : T - 1;
    constexpr int KT = BlockShape<D>::KT;
    const int keys = QW_SEG(tiles_per_split) * KT, k_begin = lo / 32 * 32 + sp * keys, k_end = min(T, k_begin + keys);
    half8 qb[NM];
    {
        const int seq = (row_base + rr) / (a.Tq * a.G), x = (row_base + rr) % (a.Tq * a.G);
        const f16* qrow = a.q + (((int64_t)seq * a.hkv * a.G + h * a.G + x % a.G) * a.Tq + x / a.G) * D + DG * g;
#pragma unroll
        for (int m = 0; m < NM; m++) {
            u32x4 w = *(const u32x4*)(qrow + 8 * m);
            if (!row_ok) w = u32x4{0, 0, 0, 0};
            if constexpr (KIND == 4)  // dims in deq4's order
                w = u32x4{__builtin_amdgcn_perm(w.z, w.x, 0x05040100u), __builtin_amdgcn_perm(w.z, w.x, 0x07060302u),
                          __builtin_amdgcn_perm(w.w, w.y, 0x05040100u), __builtin_amdgcn_perm(w.w, w.y, 0x07060302u)};
            qb[m] = as_h8(w);
        }
    }
    const uint32_t code_off = QW_SEG(code_off2);
    const int64_t krow0 = (int64_t)hc * cap + 8 * (r16 >> 2) + (r16 & 3), vblk0 = (int64_t)hc * (cap / 8) + g;
    const u32x4* const ksrc = (const u32x4*)(QW_SEG(k_data) + krow0 * (D * KIND / 32) + g * (DG * KIND / 32));
    const uint32_t* const kpsrc = KIND == 16 ? nullptr : QW_SEG(k_params) + krow0 * NG + k_param_slot(g * DG / kGroup, NG);
    const u32x4* const vsrc = (const u32x4*)(QW_SEG(v_data) + vblk0 * (D * KIND / 4)) + r16;
    const u32x4* const vpsrc =
        KIND == 16 ? nullptr : (const u32x4*)(QW_SEG(v_params) + (vblk0 * NG + r16 * DPL / kGroup) * 8);
    u32x4 kc[2][KP], vc[VP], vp[2];
    uint32_t kp[2];
    auto load_k = [&](int key) {
#pragma unroll
        for (int tt = 0; tt < 2; tt++) {
#pragma unroll
            for (int i = 0; i < KP; i++) kc[tt][i] = ksrc[(int64_t)(key + 4 * tt) * (D * KIND / 128) + i];
            if constexpr (KIND != 16) kp[tt] = kpsrc[(int64_t)(key + 4 * tt) * NG];
        }
    };
    auto load_v = [&](int key) {
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
            if constexpr (KIND != 16) {
                const half2v sb = h2(kp[tt]), s = {sb.x, sb.x}, b = {sb.y, sb.y};
                pc = make_consts<FAST, KIND>(s, s, s, s, b, b, b, b, code_off);
            }
#pragma unroll
            for (int m = 0; m < NM; m++) {
                half8 ka;
                if constexpr (KIND == 16)
                    ka = as_h8(kc[tt][m]);
                else if constexpr (KIND == 8)
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
        PairConsts pc;
        if constexpr (KIND != 16)
            pc = make_consts<FAST, KIND>(h2(vp[0][0]), h2(vp[0][1]), h2(vp[0][2]), h2(vp[0][3]), h2(vp[1][0]), h2(vp[1][1]),
                                         h2(vp[1][2]), h2(vp[1][3]), code_off);
        const u32x4 keep = keep_keys(T - (key + 8 * g)) & ~keep_keys(lo - (key + 8 * g));
#pragma unroll
        for (int j = 0; j < VP; j++) {
            half8 y[E];
#pragma unroll
            for (int i = 0; i < E; i++)
                y[i] = KIND == 16  ? as_h8(vc[j])
                       : KIND == 8 ? deq8<FAST>(vc[j][2 * i % 4], vc[j][(2 * i + 1) % 4], pc)
                                   : deq4<FAST>(vc[j][i % 4], pc, magic);
            if (edge) {  // hidden keys have weight 0, but 0 x inf is NaN
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
    static_assert((16 * kWaves * 2 + kWaves * 16 * D) * 4 <= 2 * BlockShape<D>::BUF, "the waves' sums fit the tile buffers");
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
        float* o = s_o + (wave * rows + 4 * g + e) * D + NT * r16;
#pragma unroll
        for (int c = 0; c < NT; c += 4)
            *(float4v*)(o + c) = float4v{acc_o[c][e] * fe, acc_o[c + 1][e] * fe, acc_o[c + 2][e] * fe, acc_o[c + 3][e] * fe};
    }
    __syncthreads();
    const int64_t pbase = ((int64_t)(QW_SEG(slot0) + sp) * a.hkv + h) * a.R + row_base;
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
            const int seq = (row_base + row) / (a.Tq * a.G), x = (row_base + row) % (a.Tq * a.G);
            half4v y;
#pragma unroll
            for (int j = 0; j < 4; j++) y[j] = (f16)(o[j] * inv);
            *(half4v*)(a.out + (((int64_t)seq * a.hkv * a.G + h * a.G + x % a.G) * a.Tq + x / a.G) * D + 4 * c) = y;
        } else {
            *(float4v*)(a.part_o + (pbase + row) * D + 4 * c) = o;
        }
    }
}

template <int KIND, int D, bool FAST>
__device__ __forceinline__ void unit_body(const SharedArgs& a, char* lds) {
    if (((int)blockIdx.x >= a.seg[0].n_units ? a.seg[1].rows : a.seg[0].rows) <= kFewRows)
        few_body<KIND, D, FAST>(a, lds);
    else
        shared_body<KIND, D, FAST>(a, lds);
}
#undef QW_SEG

template <int KIND, int D>
__global__ __launch_bounds__(64 * kWaves, 1) void shared_attend_kernel(SharedArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const bool fast = KIND != 16 && *((int)blockIdx.x >= a.seg[0].n_units ? a.seg[1].fast_flag : a.seg[0].fast_flag);
    if constexpr (KIND != 16)
        if (fast) return unit_body<KIND, D, true>(a, lds);
    unit_body<KIND, D, false>(a, lds);
}

template <int D>
__global__ __launch_bounds__(256) void shared_merge_kernel(SharedArgs a) {
    __shared__ SharedMerge<D> sm;
    merge_row<D>(a, blockIdx.x, blockIdx.y, sm);
}

// What a launch of a prefix and tail units costs on 256 CUs, in key tiles: prefix units of a
// tiles first, tail units of b as CUs come free.
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
    s.cap = c.cap;
    s.T = c.offset;
    s.code_off2 = c.code_offset2();
    s.fast_flag = c.fast_flag;
}

template <int KIND, int D>
int launch_units(const SharedArgs& a, hipStream_t stream) {
    const size_t shmem = (size_t)2 * BlockShape<D>::BUF;
    if (int rc = ensure_dynamic_lds((const void*)shared_attend_kernel<KIND, D>, shmem)) return rc;
    hipLaunchKernelGGL((shared_attend_kernel<KIND, D>), dim3(a.seg[0].n_units + a.seg[1].n_units),
                       dim3(64 * kWaves), shmem, stream, a);
    QW_HIP_CHECK(hipGetLastError());
    return QW_OK;
}

int launch_units(int bits, int D, const SharedArgs& a, hipStream_t stream) {
    if (a.seg[0].n_units + a.seg[1].n_units == 0) return QW_OK;
    if (D == 256)
        return bits == 4   ? launch_units<4, 256>(a, stream)
               : bits == 8 ? launch_units<8, 256>(a, stream)
                           : launch_units<16, 256>(a, stream);
    return bits == 4   ? launch_units<4, 128>(a, stream)
           : bits == 8 ? launch_units<8, 128>(a, stream)
                       : launch_units<16, 128>(a, stream);
}

}  // namespace

int plan_shared(const KVCache* prefix, const KVCache* tails, const void* q, int n_seq, int n_rows, int G, int hkv,
                const int32_t* starts, float scale, bool causal, void* out, hipStream_t stream, SharedArgs* pa) {
    SharedArgs& a = *pa;
    a = SharedArgs{};
    const KVCache* c[2] = {prefix && prefix->offset > 0 ? prefix : nullptr, tails && tails->offset > 0 ? tails : nullptr};
    const int D = (prefix ? prefix : tails)->D, KT = 16384 / D;
    a.q = (const f16*)q;
    a.out = (f16*)out;
    a.starts = starts;
    a.Tq = n_rows;
    a.G = G;
    a.hkv = hkv;
    a.R = n_seq * n_rows * G;
    a.scale2 = scale * kLog2e;
    int tiles[2] = {0, 0}, n_qt[2] = {0, 0};
    for (int i = 0; i < 2; i++) {
        SharedSegment& s = a.seg[i];
        s.n_split = s.heads = 1;
        if (!c[i]) continue;
        fill_cache(s, *c[i]);
        s.heads = c[i]->hkv;
        s.rows = i == 0 ? a.R : n_rows * G;
        const int rt = (s.rows + 15) / 16;
        n_qt[i] = (rt + kWaves - 1) / kWaves;
        s.unit_rows = 16 * ((rt + n_qt[i] - 1) / n_qt[i]);
        s.causal_rows = i == 1 && causal ? n_rows : 0;
        tiles[i] = (s.T + KT - 1) / KT;
    }
    // Tiles a split: the count with the shortest launch (a unit's prologue and partials cost
    // about two tiles, a partial row read again by the merge a share of one).
    const int most = std::max(tiles[0], tiles[1]);
    const int64_t u0 = (int64_t)n_qt[0] * a.seg[0].heads, u1 = (int64_t)n_qt[1] * a.seg[1].heads;
    int best = most;
    double best_cost = 1e30;
    for (int tps = 1; tps <= most; tps += std::max(1, tps / 16)) {
        const int s0 = (tiles[0] + tps - 1) / tps, s1 = (tiles[1] + tps - 1) / tps;
        if (s0 + s1 > kSharedMaxSlots) continue;
        const double cost = makespan(u0 * s0, std::min(tps, tiles[0]) + 2.0, u1 * s1, std::min(tps, tiles[1]) + 2.0) +
                            (s0 + s1) * (double)a.R * hkv * D * 2e-7;
        if (cost < best_cost) {
            best_cost = cost;
            best = tps;
        }
    }
    a.n_slots = 0;
    for (int i = 0; i < 2; i++) {
        SharedSegment& s = a.seg[i];
        if (!c[i]) continue;
        s.tiles_per_split = best;
        s.n_split = (tiles[i] + best - 1) / best;
        s.slot0 = a.n_slots;
        a.n_slots += s.n_split;
        const int64_t units = (int64_t)n_qt[i] * s.heads * s.n_split;
        QW_REQUIRE(units < (int64_t)1 << 30, QW_ERR_UNSUPPORTED, "shared attention: too many rows for one call");
        s.n_units = (int)units;
    }
    const size_t rows = (size_t)a.n_slots * hkv * a.R;
    const size_t o_bytes = a.n_slots > 1 ? rows * D * sizeof(float) : 0;
    void* ws = nullptr;
    if (int rc = workspace(kWsShared, (prefix ? prefix : tails)->device, stream, o_bytes + rows * sizeof(float2), &ws))
        return rc;
    a.part_o = (float*)ws;
    a.part_ml = (float2*)((char*)ws + o_bytes);
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
    if (D == 256)
        hipLaunchKernelGGL(shared_merge_kernel<256>, dim3(a.R, a.hkv), dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL(shared_merge_kernel<128>, dim3(a.R, a.hkv), dim3(256), 0, stream, a);
    QW_HIP_CHECK(hipGetLastError());
    return QW_OK;
}

static int check_shared(const KVCache& p, const KVCache* t, int n_seq, const void* q, int n_q_heads, int n_rows,
                        float scale, const void* out, int tail_rows) {
    QW_REQUIRE(q && out, QW_ERR_INVALID_ARGUMENT, "shared attention: null q/out");
    QW_REQUIRE(n_seq > 0 && n_rows > 0 && n_q_heads > 0 && n_q_heads % p.hkv == 0, QW_ERR_INVALID_ARGUMENT,
               "shared attention: n_seq, n_rows > 0 and n_q_heads a positive multiple of n_kv_heads");
    QW_REQUIRE((int64_t)n_seq * n_rows * (n_q_heads / p.hkv) <= INT32_MAX / 2, QW_ERR_INVALID_ARGUMENT,
               "shared attention: too many rows");
    QW_REQUIRE(std::isfinite(scale), QW_ERR_INVALID_ARGUMENT, "shared attention: scale must be finite");
    QW_REQUIRE(!p.turbo4() && !(t && t->turbo4()), QW_ERR_UNSUPPORTED, "shared attention: not over Turbo4 caches");
    if (t) {
        QW_REQUIRE(t != &p, QW_ERR_INVALID_ARGUMENT, "shared attention: the prefix and the tails are one cache");
        QW_REQUIRE((int64_t)n_seq * p.hkv == t->hkv && t->D == p.D && t->device == p.device, QW_ERR_INVALID_ARGUMENT,
                   "shared attention: the tails need n_seq * n_kv_heads heads of the prefix's head_dim, on its device");
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
    const int tail_rows = tails ? tails->offset + (append ? n_rows : 0) : 0;
    if (int rc = check_shared(prefix, tails, n_seq, q, n_q_heads, n_rows, scale, out, tail_rows)) return rc;
    DeviceGuard dg(prefix.device);
    QW_REQUIRE(dg.ok, QW_ERR_HIP, "shared attention: hipSetDevice failed");
    if (append)
        if (int rc = tails->update(k_new, v_new, n_rows, stream)) return rc;
    SharedArgs a;
    if (int rc = plan_shared(&prefix, tails, q, n_seq, n_rows, n_q_heads / prefix.hkv, prefix.hkv, starts, scale, true,
                             out, stream, &a))
        return rc;
    if (int rc = launch_shared(&prefix, tails, a, stream)) return rc;
    return launch_shared_merge(prefix.D, a, stream);
}

}  // namespace qw
