// key_weights.hip - attention over a cache that also counts what weight each key
// got, gfx950.
//
// For row r and query head j of KV head h, p[j][r][t] = softmax over the visible t of
// scale q . k_t (the attention of attend_shared.hip over one cache), and
//   weights_out[h][t] = decay weights[h][t] + sum over j of the group, r of p[j][r][t].
// The reference's runtime has no such call; its caches only grow (KVCache::update,
// crates/mlxcel-core/src/cache.rs:922) or are trimmed at the end (:2251).
//
// p needs the row's whole sum, so K is seen twice: the attention launch leaves each row's
// maximum and sum, and key_weights_kernel forms the scores again. A wave owns 32 keys: it
// dequantizes their K rows once, into registers as the A operand of S^T = K . Q^T, and runs
// over the row tiles; a lane keeps its 8 keys' sums over its rows in fp32 and 16 lanes add
// theirs up at the end. Every key belongs to one wave: no atomics, the same bits each time.
#include <algorithm>
#include <cmath>

#include "attend_shared.hpp"
#include "dequant.hpp"

namespace qw {

namespace {

struct WeightArgs {
    SharedArgs s;            // seg[1]: the cache
    const float2* row_ml;    // [hkv][R]: the row's maximum (log2 units) and 1 / its sum
    const float* weights;    // [hkv][ws_in] or null
    float* weights_out;      // [hkv][ws_out]
    int64_t ws_in, ws_out;
    int n_weights;           // keys that weights covers
    float decay;
};

// A row's maximum and 1 / sum over its partials (apart: one logarithm of the sum would round
// at the maximum's size): grid (R / 4, hkv), a wave a row.
__global__ __launch_bounds__(256) void row_sums_kernel(SharedArgs a, float2* __restrict__ row_ml) {
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6), h = blockIdx.y, lane = threadIdx.x & 63;
    if (row >= a.R) return;
    const int64_t stride = (int64_t)a.hkv * a.R, at = (int64_t)h * a.R + row;
    float M = -INFINITY;
    for (int s = lane; s < a.n_slots; s += 64) M = fmaxf(M, a.part_ml[s * stride + at].x);
    M = wave_reduce(M, OpMax{});
    const float mr = M == -INFINITY ? 0.0f : M;
    float l = 0.0f;
    for (int s = lane; s < a.n_slots; s += 64) {
        const float2 ml = a.part_ml[s * stride + at];
        l += __builtin_amdgcn_exp2f(ml.x - mr) * ml.y;
    }
    l = wave_reduce(l, OpSum{});
    if (lane == 0) row_ml[at] = float2{mr, l == 0.0f ? 0.0f : 1.0f / l};
}

template <int KIND, int D>
__global__ __launch_bounds__(256) void key_weights_kernel(WeightArgs w) {
    constexpr int NM = D / 32, NG = D / kGroup, DG = D / 4;  // DG: dims of a lane group
    const SharedSegment& c = w.s.seg[1];
    const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4, h = blockIdx.y;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int key0 = (blockIdx.x * 4 + wave) * 32, T = c.T;
    if (key0 >= T) return;
    const uint32_t magic = vconst(kMagic);
    // A operand: lane (g, r16) holds dims DG g .. + DG - 1 of key 8 (r16 >> 2) + 4 tt + (r16 & 3),
    // so that a lane of S^T gets keys 8 g + e of row r16
    half8 ka[2][NM];
#pragma unroll
    for (int tt = 0; tt < 2; tt++) {
        const int64_t row = (int64_t)h * c.cap + key0 + 8 * (r16 >> 2) + 4 * tt + (r16 & 3);
        const u32x4* src = (const u32x4*)(c.k_data + row * (D * KIND / 32) + g * (DG * KIND / 32));
        u32x4 x[DG * KIND / 128];
#pragma unroll
        for (int u = 0; u < DG * KIND / 128; u++) x[u] = src[u];
        if constexpr (KIND == 16) {
#pragma unroll
            for (int m = 0; m < NM; m++) ka[tt][m] = as_h8(x[m]);
        } else {
            const half2v sb = h2(c.k_params[row * NG + k_param_slot(g * DG / kGroup, NG)]);
            const half2v s = {sb.x, sb.x}, b = {sb.y, sb.y};
            const PairConsts pc = make_consts<false, KIND>(s, s, s, s, b, b, b, b, c.code_off2);
#pragma unroll
            for (int m = 0; m < NM; m++)
                ka[tt][m] = KIND == 4 ? deq4<false>(x[m / 4][m % 4], pc, magic)
                                      : deq8<false>(x[m * KIND / 16 % (DG * KIND / 128)][2 * m % 4],
                                                    x[m * KIND / 16 % (DG * KIND / 128)][2 * m % 4 + 1], pc);
        }
    }
    const int G = w.s.G, Tq = w.s.Tq, R = w.s.R;
    auto limit = [&](int row) { return c.causal_rows ? T - c.causal_rows + row / G : T - 1; };
    // the first row tile with a row that sees key0
    const int first = c.causal_rows ? max(0, key0 - (T - c.causal_rows)) * G / 16 * 16 : 0;
    float sum[8] = {};
    for (int row0 = first; row0 < R; row0 += 16) {
        const int row = row0 + r16, rr = min(row, R - 1);
        const f16* qrow = w.s.q + ((int64_t)(h * G + rr % G) * Tq + rr / G) * D + DG * g;
        const float2 ml = w.row_ml[(int64_t)h * R + rr];
        half8 qb[NM];
#pragma unroll
        for (int m = 0; m < NM; m++) {
            u32x4 x = *(const u32x4*)(qrow + 8 * m);
            if constexpr (KIND == 4)  // dims in the order of deq4
                x = u32x4{__builtin_amdgcn_perm(x.z, x.x, 0x05040100u), __builtin_amdgcn_perm(x.z, x.x, 0x07060302u),
                          __builtin_amdgcn_perm(x.w, x.y, 0x05040100u), __builtin_amdgcn_perm(x.w, x.y, 0x07060302u)};
            qb[m] = as_h8(x);
        }
        float4v acc[2] = {float4v{0.f, 0.f, 0.f, 0.f}, float4v{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int m = 0; m < NM; m++) {
            acc[0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[0][m], qb[m], acc[0], 0, 0, 0);
            acc[1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[1][m], qb[m], acc[1], 0, 0, 0);
        }
        const int lim = limit(rr);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float p = __builtin_amdgcn_exp2f(acc[e >> 2][e & 3] * w.s.scale2 - ml.x) * ml.y;
            if (key0 + 8 * g + e <= lim && row < R) sum[e] += p;
        }
    }
#pragma unroll
    for (int e = 0; e < 8; e++) {
        float x = sum[e];
        x += lane_xor<1>(x, lane);
        x += lane_xor<2>(x, lane);
        x += lane_xor<4>(x, lane);
        x += lane_xor<8>(x, lane);
        const int key = key0 + 8 * g + e;
        if (r16 == e && key < T) {
            if (w.weights && key < w.n_weights) x += w.decay * w.weights[h * w.ws_in + key];
            w.weights_out[h * w.ws_out + key] = x;
        }
    }
}

template <int KIND, int D>
int launch_weights(const WeightArgs& w, hipStream_t stream) {
    hipLaunchKernelGGL((key_weights_kernel<KIND, D>), dim3((w.s.seg[1].T + 127) / 128, w.s.hkv), dim3(256), 0, stream, w);
    QW_HIP_CHECK(hipGetLastError());
    return QW_OK;
}

}  // namespace

int attention_scored(KVCache& c, const void* q, int n_q_heads, int n_rows, const void* k_new, const void* v_new,
                     float scale, bool causal, const float* weights, int64_t weights_stride, int n_weights,
                     float decay, float* weights_out, int64_t weights_out_stride, void* out, hipStream_t stream) {
    const bool append = k_new || v_new;
    QW_REQUIRE(q && out && weights_out, QW_ERR_INVALID_ARGUMENT, "scored attention: null q/out/weights_out");
    QW_REQUIRE(!append || (k_new && v_new), QW_ERR_INVALID_ARGUMENT, "scored attention: an append needs k_new and v_new");
    QW_REQUIRE(n_rows > 0 && n_q_heads > 0 && n_q_heads % c.hkv == 0, QW_ERR_INVALID_ARGUMENT,
               "scored attention: n_rows > 0 and n_q_heads a positive multiple of n_kv_heads");
    QW_REQUIRE((int64_t)n_rows * (n_q_heads / c.hkv) <= INT32_MAX / 32, QW_ERR_INVALID_ARGUMENT,
               "scored attention: too many rows");
    QW_REQUIRE(std::isfinite(scale) && std::isfinite(decay) && decay >= 0.0f, QW_ERR_INVALID_ARGUMENT,
               "scored attention: scale must be finite, decay finite and >= 0");
    QW_REQUIRE(!c.turbo4(), QW_ERR_UNSUPPORTED, "scored attention: not over Turbo4 caches");
    const int64_t T = (int64_t)c.offset + (append ? n_rows : 0);
    QW_REQUIRE(T > 0 && (!causal || T >= n_rows), QW_ERR_INVALID_ARGUMENT,
               "scored attention: empty cache, or fewer cached keys than causal query rows");
    QW_REQUIRE(weights_out_stride >= T && (!weights || (n_weights >= 0 && weights_stride >= n_weights)),
               QW_ERR_INVALID_ARGUMENT, "scored attention: a weights stride below its row's length");
    if (weights && decay > 0.0f && !(weights == weights_out && weights_stride == weights_out_stride)) {
        const uintptr_t a0 = (uintptr_t)weights, a1 = a0 + 4 * ((uint64_t)(c.hkv - 1) * weights_stride + n_weights);
        const uintptr_t b0 = (uintptr_t)weights_out, b1 = b0 + 4 * ((uint64_t)(c.hkv - 1) * weights_out_stride + T);
        QW_REQUIRE(a1 <= b0 || b1 <= a0, QW_ERR_INVALID_ARGUMENT,
                   "scored attention: weights_out overlaps weights and is not the same array");
    }
    DeviceGuard dg(c.device);
    QW_REQUIRE(dg.ok, QW_ERR_HIP, "scored attention: hipSetDevice failed");
    if (append)
        if (int rc = c.update(k_new, v_new, n_rows, stream)) return rc;
    WeightArgs w;
    if (int rc = plan_shared(nullptr, &c, q, 1, n_rows, n_q_heads / c.hkv, c.hkv, nullptr, scale, causal, out, stream, &w.s))
        return rc;
    void* row_ml = nullptr;
    if (int rc = workspace(kWsRowSums, c.device, stream, (size_t)c.hkv * w.s.R * sizeof(float2), &row_ml)) return rc;
    if (int rc = launch_shared(nullptr, &c, w.s, stream)) return rc;
    if (int rc = launch_shared_merge(c.D, w.s, stream)) return rc;
    w.row_ml = (const float2*)row_ml;
    w.weights = decay > 0.0f ? weights : nullptr;
    w.weights_out = weights_out;
    w.ws_in = weights_stride;
    w.ws_out = weights_out_stride;
    w.n_weights = n_weights;
    w.decay = decay;
    hipLaunchKernelGGL(row_sums_kernel, dim3((w.s.R + 3) / 4, c.hkv), dim3(256), 0, stream, w.s, (float2*)row_ml);
    QW_HIP_CHECK(hipGetLastError());
    if (c.D == 256)
        return c.bits == 4   ? launch_weights<4, 256>(w, stream)
               : c.bits == 8 ? launch_weights<8, 256>(w, stream)
                             : launch_weights<16, 256>(w, stream);
    return c.bits == 4   ? launch_weights<4, 128>(w, stream)
           : c.bits == 8 ? launch_weights<8, 128>(w, stream)
                         : launch_weights<16, 128>(w, stream);
}

}  // namespace qw
