// key_weights.hip - attention over a cache that also counts what weight each key
// got, gfx950.
//
// For row r and query head j of KV head h, p[j][r][t] = softmax over the visible t of
// scale q . k_t (the attention of attend_shared.hip over one cache), and
//   weights_out[h][t] = decay weights[h][t] + sum over j of the group, r of p[j][r][t].
// The reference's runtime has no such call; its caches only grow (KVCache::update,
// crates/mlxcel-core/src/cache.rs:922) or are trimmed at the end (:2251).
//
// p needs the row's whole sum. Up to 16 rows a KV head the attention launch keeps its scores
// (4 bytes a row and key, where K again would be 144 to 512 a key) and finish_few_kernel turns them
// into weights beside the merge (one row over 32k 4-bit keys: 14.4 + 4.9 us, of which the
// keys themselves at 4.98 TB/s are 7.8). For more rows K is seen twice: the attention launch leaves each
// row's maximum and sum, and key_weights_kernel forms the scores again. A wave owns 64 keys: it
// dequantizes their K rows once, into registers as the A operand of S^T = K . Q^T, and runs
// over the rows, 32 a step, whose q the workgroup's 8 waves share through LDS (LDS-DMA, the next
// step's while this one computes). A lane keeps its 16 keys' sums over its rows in fp32 and 16
// lanes add theirs up at the end. Where the keys alone leave CUs idle the rows are split too, each
// split's sums to a workspace, added up in order: no atomics, the same bits each time.
// Bound by the MFMAs and the exponentials beside them (a product-and-sum, an exponential and a
// product-and-sum a weight): 1536 rows over 9.7k Int8 keys, D = 256, 236 us, 0.72 PFLOP/s, the MFMAs busy
// 0.35 of the profiler's window; K formed again for each step of rows took 1050 us a call. A wave's K takes 128 of
// some 212 registers at D = 256; over Turbo4 keys the lookups beside them spill 36.
#include <algorithm>
#include <cmath>

#include "attend_shared.hpp"
#include "dequant.hpp"
#include "turbo4_device.hpp"

namespace qw {

namespace {

struct WeightArgs {
    SharedArgs s;            // seg[1]: the cache
    const float* weights;    // [hkv][ws_in] or null
    float* weights_out;      // [hkv][ws_out]
    float* part;             // [row_splits][hkv][T] where the rows are split
    int64_t ws_in, ws_out;
    int n_weights;           // keys that weights covers
    float decay;
    float scale2;            // scale * log2 e, with its sign (the attention launch takes q negated instead)
    int row_splits, rows_per_split;  // (rows_per_split a multiple of kStepRows)
};

constexpr int kWaveKeys = 64, kWgWaves = 8, kWgKeys = kWaveKeys * kWgWaves, kStepRows = 32;

__device__ __forceinline__ void store_weight(const WeightArgs& w, int h, int key, float x) {
    if (w.weights && key < w.n_weights) x += w.decay * w.weights[h * w.ws_in + key];
    w.weights_out[h * w.ws_out + key] = x;
}

// A row's maximum and 1 / sum (apart: one logarithm of the sum would round at the maximum's size)
// where one slot holds it and no merge runs: a thread a row, grid (R / 256, hkv).
__global__ __launch_bounds__(256) void row_sums_kernel(SharedArgs a) {
    const int row = blockIdx.x * 256 + threadIdx.x;
    if (row >= a.R) return;
    const int64_t at = (int64_t)blockIdx.y * a.R + row;
    const float2 ml = a.part_ml[at];
    a.row_ml[at] = float2{ml.x == -INFINITY ? 0.0f : ml.x, ml.y == 0.0f ? 0.0f : 1.0f / ml.y};
}

template <int KIND, int D, bool T4>
__global__ __launch_bounds__(64 * kWgWaves) void key_weights_kernel(WeightArgs w) {
    constexpr int NM = D / 32, NG = D / kGroup, E = 16 / KIND;
    constexpr int TILE = D * 2 * 16;                         // bytes of 16 rows of q
    constexpr int KP = D * KIND / 512;                       // 16-byte pieces of a K row a lane group
    __shared__ __attribute__((aligned(16))) char lds[2][2 * TILE];  // [buffer][row tile][D / 8 chunks][16 rows]
    const SharedSegment& c = w.s.seg[1];
    const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4, h = blockIdx.y;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int T = c.T, G = w.s.G, Tq = w.s.Tq, R = w.s.R;
    const int key0 = blockIdx.x * kWgKeys + wave * kWaveKeys;
    const bool live = key0 < T;
    const uint32_t magic = vconst(kMagic);
    __shared__ float2 cp[T4 ? 256 : 1];  // Turbo4: the centroids of a byte of indices
    if constexpr (T4) {
        if (tid < 256) cp[tid] = float2{c.t4_cb[tid & 15], c.t4_cb[tid >> 4]};
        __syncthreads();
    }
    // A operands: lane (g, r16) holds its pieces (k_chunk) of key 32 u + 8 (r16 >> 2) + 4 tt + (r16 &
    // 3), so that a lane of S^T gets keys 32 u + 8 g + e of row r16
    half8 ka[2][2][NM];
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
        for (int tt = 0; tt < 2; tt++) {
            const int key = min(key0 + 32 * u + 8 * (r16 >> 2) + 4 * tt + (r16 & 3), c.cap - 1);
            const int64_t row = (int64_t)h * c.cap + key;
            const u32x4* src = (const u32x4*)(c.k_data + row * (D * KIND / 32)) + g;
            u32x4 x[KP];
#pragma unroll
            for (int i = 0; i < KP; i++) x[i] = src[4 * i];
            if constexpr (KIND == 16) {
#pragma unroll
                for (int m = 0; m < NM; m++) ka[u][tt][m] = as_h8(x[m]);
            } else if constexpr (T4) {
                const float kr = (float)h2(c.k_params[row]).x;
#pragma unroll
                for (int m = 0; m < NM; m++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float2 y = cp[x[m / 4][m % 4] >> (8 * i) & 0xFFu];
                        ka[u][tt][m][2 * i] = t4_f16_product(y.x, kr);
                        ka[u][tt][m][2 * i + 1] = t4_f16_product(y.y, kr);
                    }
            } else {
                uint32_t kp[KP];
#pragma unroll
                for (int i = 0; i < KP; i++) kp[i] = c.k_params[row * NG + k_param_slot(k_piece_group<KIND>(i, g), NG)];
#pragma unroll
                for (int m = 0; m < NM; m++) {
                    const half2v sb = h2(kp[m / E]), s = {sb.x, sb.x}, b = {sb.y, sb.y};
                    const PairConsts pc = make_consts<false, KIND>(s, s, s, s, b, b, b, b, c.code_off2);
                    if constexpr (KIND == 4) {  // dims come as pairs (0,4), (1,5), (2,6), (3,7)
                        const u32x4 y = __builtin_bit_cast(u32x4, deq4<false>(x[m / 4][m % 4], pc, magic));
                        ka[u][tt][m] = as_h8(u32x4{__builtin_amdgcn_perm(y.y, y.x, 0x05040100u),
                                                   __builtin_amdgcn_perm(y.w, y.z, 0x05040100u),
                                                   __builtin_amdgcn_perm(y.y, y.x, 0x07060302u),
                                                   __builtin_amdgcn_perm(y.w, y.z, 0x07060302u)});
                    } else {
                        ka[u][tt][m] = deq8<false>(x[m / 2][2 * m % 4], x[m / 2][2 * m % 4 + 1], pc);
                    }
                }
            }
        }
    auto limit = [&](int row) { return c.causal_rows ? T - c.causal_rows + row / G : T - 1; };
    // rows: the split's, from the first step that holds a row which sees the workgroup's first key
    const int wg_key0 = blockIdx.x * kWgKeys;
    const int first = c.causal_rows ? max(0, wg_key0 - (T - c.causal_rows)) * G : 0;
    const int row_end = min(R, ((int)blockIdx.z + 1) * w.rows_per_split);
    const int row_begin = max((int)blockIdx.z * w.rows_per_split, first / kStepRows * kStepRows);
    // q of 32 rows into a buffer: wave i copies chunks 4 j .. + 3 of both row tiles for j = i, i + 8, ..
    const uint32_t lds0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)&lds[0][0];
    auto dma = [&](int row0, int buf) {
#pragma unroll
        for (int i = 0; i < 2 * (D / 32) / kWgWaves; i++) {
            const int j = wave + kWgWaves * i, rt = j / (D / 32), c4 = j % (D / 32);
            const int row = min(row0 + 16 * rt + r16, R - 1), r = row / G;
            const f16* src = w.s.q + ((int64_t)(h * G + row - r * G) * Tq + r) * D + 8 * (4 * c4 + g);
            uint32_t saved;
            asm volatile(
                "s_mov_b32 %0, m0\n\t"
                "s_mov_b32 m0, %2\n\t"
                "s_nop 0\n\t"
                "global_load_lds_dwordx4 %1, off\n\t"
                "s_nop 0\n\t"
                "s_mov_b32 m0, %0"
                : "=&s"(saved)
                : "v"(src), "s"(__builtin_amdgcn_readfirstlane(lds0 + buf * 2 * TILE + rt * TILE + c4 * 1024))
                : "memory");
        }
    };
    auto stats = [&](int row) {  // (a row past the last: weights of 2^-inf times 0)
        const float2 ml = w.s.row_ml[(int64_t)h * R + min(row, R - 1)];
        return row < R ? ml : float2{INFINITY, 0.0f};
    };
    float sum[2][8] = {};
    float2 ml[2], ml_next[2] = {};
    if (row_begin < row_end) {
        dma(row_begin, 0);
#pragma unroll
        for (int rt = 0; rt < 2; rt++) ml_next[rt] = stats(row_begin + 16 * rt + r16);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    for (int row0 = row_begin; row0 < row_end; row0 += kStepRows) {
        const int buf = (row0 - row_begin) / kStepRows & 1;
#pragma unroll
        for (int rt = 0; rt < 2; rt++) ml[rt] = ml_next[rt];
        if (row0 + kStepRows < row_end) {
            dma(row0 + kStepRows, buf ^ 1);
#pragma unroll
            for (int rt = 0; rt < 2; rt++) ml_next[rt] = stats(row0 + kStepRows + 16 * rt + r16);
        }
        if (live) {
#pragma unroll
            for (int rt = 0; rt < 2; rt++) {
                const half8* q8 = (const half8*)(lds[buf] + rt * TILE) + E * 16 * g + r16;
                float4v acc[2][2];
#pragma unroll
                for (int u = 0; u < 2; u++) acc[u][0] = acc[u][1] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int m = 0; m < NM; m++) {
                    const half8 qb = q8[16 * k_chunk<KIND>(m, 0)];
#pragma unroll
                    for (int u = 0; u < 2; u++)
#pragma unroll
                        for (int tt = 0; tt < 2; tt++)
                            acc[u][tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[u][tt][m], qb, acc[u][tt], 0, 0, 0);
                }
                auto weight = [&](int u, int e) {
                    return __builtin_amdgcn_exp2f(__builtin_fmaf(acc[u][e >> 2][e & 3], w.scale2, -ml[rt].x));
                };
                // the tile's first row's limit decides whether any key of the wave is hidden in it
                if (limit(row0 + 16 * rt) < key0 + kWaveKeys - 1) {
                    const int lim = limit(row0 + 16 * rt + r16);
#pragma unroll
                    for (int u = 0; u < 2; u++)
#pragma unroll
                        for (int e = 0; e < 8; e++)
                            if (key0 + 32 * u + 8 * g + e <= lim) sum[u][e] = __builtin_fmaf(weight(u, e), ml[rt].y, sum[u][e]);
                } else {
#pragma unroll
                    for (int u = 0; u < 2; u++)
#pragma unroll
                        for (int e = 0; e < 8; e++) sum[u][e] = __builtin_fmaf(weight(u, e), ml[rt].y, sum[u][e]);
                }
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    }
    if (!live) return;
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
            float x = sum[u][e];
            x += lane_xor<1>(x, lane);
            x += lane_xor<2>(x, lane);
            x += lane_xor<4>(x, lane);
            x += lane_xor<8>(x, lane);
            const int key = key0 + 32 * u + 8 * g + e;
            if (r16 != e + 8 * u || key >= T) continue;
            if (w.row_splits > 1)
                w.part[((int64_t)blockIdx.z * w.s.hkv + h) * T + key] = x;
            else
                store_weight(w, h, key, x);
        }
}

__global__ __launch_bounds__(256) void copy_halves_kernel(const f16* __restrict__ from, f16* __restrict__ to, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) to[i] = from[i];
}

// The row splits' sums, in order.
__global__ __launch_bounds__(256) void add_weights_kernel(WeightArgs w) {
    const int T = w.s.seg[1].T, key = blockIdx.x * 256 + threadIdx.x, h = blockIdx.y;
    if (key >= T) return;
    float x = 0.0f;
    for (int i = 0; i < w.row_splits; i++) x += w.part[((int64_t)i * w.s.hkv + h) * T + key];
    store_weight(w, h, key, x);
}

// Few rows (the attention launch kept their scores): the rows merged by the first workgroups of
// a head and the keys' weights formed by the others, 1024 keys each, from the scores and the rows'
// statistics, which every one of them joins for itself.
template <int D>
__global__ __launch_bounds__(256) void finish_few_kernel(WeightArgs w, int n_merge) {
    __shared__ SharedMerge sm;
    __shared__ float2 s_ml[16];
    const int h = blockIdx.y, tid = threadIdx.x, R = w.s.R, T = w.s.seg[1].T;
    if ((int)blockIdx.x < n_merge) {
        merge_group<D>(w.s, blockIdx.x, h, sm);
        return;
    }
    {
        const int row = min(tid / 16, R - 1), i16 = tid % 16;  // 16 lanes a row
        const int64_t stride = (int64_t)w.s.hkv * R, at = (int64_t)h * R + row;
        float M = -INFINITY, l = 0.0f;
        for (int s = i16; s < w.s.n_slots; s += 16) M = fmaxf(M, w.s.part_ml[s * stride + at].x);
        const int lane = tid & 63;
        M = fmaxf(M, lane_xor<1>(M, lane));
        M = fmaxf(M, lane_xor<2>(M, lane));
        M = fmaxf(M, lane_xor<4>(M, lane));
        M = fmaxf(M, lane_xor<8>(M, lane));
        const float mr = M == -INFINITY ? 0.0f : M;
        for (int s = i16; s < w.s.n_slots; s += 16) {
            const float2 ml = w.s.part_ml[s * stride + at];
            l += __builtin_amdgcn_exp2f(ml.x - mr) * ml.y;
        }
        l += lane_xor<1>(l, lane);
        l += lane_xor<2>(l, lane);
        l += lane_xor<4>(l, lane);
        l += lane_xor<8>(l, lane);
        if (i16 == 0) s_ml[tid / 16] = float2{mr, l == 0.0f ? 0.0f : 1.0f / l};
    }
    __syncthreads();
    const int key = ((int)blockIdx.x - n_merge) * 1024 + 4 * tid;
    if (key >= T) return;
    const int causal = w.s.seg[1].causal_rows, first_lim = causal ? T - causal : T - 1;
    float sum[4] = {};
    const float* sc = w.s.scores + (int64_t)h * R * w.s.score_stride + key;
    for (int row = 0; row < R; row++) {
        const float4v s = *(const float4v*)(sc + row * w.s.score_stride);
        const float2 ml = s_ml[row];
        const int lim = causal ? first_lim + row / w.s.G : first_lim;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float p = __builtin_amdgcn_exp2f(s[e] - ml.x) * ml.y;
            sum[e] += key + e <= lim ? p : 0.0f;
        }
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (key + e < T) store_weight(w, h, key + e, sum[e]);
}

template <int KIND, int D, bool T4 = false>
int launch_weights(const WeightArgs& w, hipStream_t stream) {
    const int T = w.s.seg[1].T;
    hipLaunchKernelGGL((key_weights_kernel<KIND, D, T4>), dim3((T + kWgKeys - 1) / kWgKeys, w.s.hkv, w.row_splits),
                       dim3(64 * kWgWaves), 0, stream, w);
    QW_HIP_CHECK(hipGetLastError());
    if (w.row_splits > 1) {
        hipLaunchKernelGGL(add_weights_kernel, dim3((T + 255) / 256, w.s.hkv), dim3(256), 0, stream, w);
        QW_HIP_CHECK(hipGetLastError());
    }
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
    const int64_t T = (int64_t)c.offset + (append ? n_rows : 0);
    QW_REQUIRE(T > 0 && (!causal || T >= n_rows), QW_ERR_INVALID_ARGUMENT,
               "scored attention: empty cache, or fewer cached keys than causal query rows");
    QW_REQUIRE(weights_out_stride >= T && (!weights || (n_weights >= 0 && weights_stride >= n_weights)),
               QW_ERR_INVALID_ARGUMENT, "scored attention: a weights stride below its row's length");
    if (weights && decay > 0.0f && !(weights == weights_out && (weights_stride == weights_out_stride || c.hkv == 1))) {
        const uintptr_t a0 = (uintptr_t)weights, a1 = a0 + 4 * ((uint64_t)(c.hkv - 1) * weights_stride + n_weights);
        const uintptr_t b0 = (uintptr_t)weights_out, b1 = b0 + 4 * ((uint64_t)(c.hkv - 1) * weights_out_stride + T);
        QW_REQUIRE(a1 <= b0 || b1 <= a0, QW_ERR_INVALID_ARGUMENT,
                   "scored attention: weights_out overlaps weights and is not the same array");
    }
    DeviceGuard dg(c.device);
    QW_REQUIRE(dg.ok, QW_ERR_HIP, "scored attention: hipSetDevice failed");
    // (what can fail for want of memory comes before the append)
    if (append)
        if (int rc = make_room(c, n_rows, stream)) return rc;
    WeightArgs w;
    if (int rc = plan_shared(nullptr, &c, (int)T, q, 1, n_rows, n_q_heads / c.hkv, c.hkv, nullptr, scale, causal, out, stream,
                             &w.s))
        return rc;
    const int R = w.s.R;
    const int64_t q_rows = (int64_t)n_q_heads * n_rows;
    const bool t4 = c.turbo4();
    if (t4)
        if (int rc = shared_turbo4_room(c, q_rows, stream, &w.s)) return rc;
    w.weights = decay > 0.0f ? weights : nullptr;
    w.weights_out = weights_out;
    w.ws_in = weights_stride;
    w.ws_out = weights_out_stride;
    w.n_weights = n_weights;
    w.decay = decay;
    w.scale2 = w.s.q_flip ? -w.s.scale2 : w.s.scale2;
    if (R <= 16) {
        w.s.score_stride = (T + 31) / 32 * 32;
        void* scores = nullptr;
        if (int rc = workspace(kWsRowSums, c.device, stream, (size_t)c.hkv * R * w.s.score_stride * sizeof(float), &scores))
            return rc;
        w.s.scores = (float*)scores;
        if (append)
            if (int rc = c.update(k_new, v_new, n_rows, stream)) return rc;
        if (t4)
            if (int rc = shared_turbo4_rotate_q(c, q, q_rows, w.s, stream)) return rc;
        if (int rc = launch_shared(nullptr, &c, w.s, stream)) return rc;
        const int n_merge = w.s.n_slots > 1 ? merge_groups(c.D, R, c.hkv, w.s.n_slots) : 0;
        const dim3 grid((unsigned)(n_merge + (T + 1023) / 1024), c.hkv);
        if (c.D == 256)
            hipLaunchKernelGGL(finish_few_kernel<256>, grid, dim3(256), 0, stream, w, n_merge);
        else
            hipLaunchKernelGGL(finish_few_kernel<128>, grid, dim3(256), 0, stream, w, n_merge);
        QW_HIP_CHECK(hipGetLastError());
        return t4 ? launch_turbo4_rotate(c, w.s.out, (int)q_rows, true, (f16*)out, stream) : QW_OK;
    }
    // row splits: about one workgroup a CU, of at least four steps each
    const int64_t groups = (T + kWgKeys - 1) / kWgKeys * c.hkv, steps = (R + kStepRows - 1) / kStepRows;
    w.row_splits = (int)std::max<int64_t>(1, std::min<int64_t>({256 / groups, steps / 4, 64}));
    w.rows_per_split = (int)((steps + w.row_splits - 1) / w.row_splits * kStepRows);
    w.row_splits = (R + w.rows_per_split - 1) / w.rows_per_split;
    const size_t ml_bytes = ((size_t)c.hkv * R * sizeof(float2) + 15) / 16 * 16;
    const size_t part_bytes = w.row_splits > 1 ? ((size_t)w.row_splits * c.hkv * T * sizeof(float) + 15) / 16 * 16 : 0;
    // the weights' kernel copies q into LDS by pieces of 16 bytes: a q off their alignment is copied first
    const size_t q_bytes = (uintptr_t)w.s.q % 16 ? (size_t)n_q_heads * n_rows * c.D * sizeof(f16) : 0;
    void* ws = nullptr;
    if (int rc = workspace(kWsRowSums, c.device, stream, ml_bytes + part_bytes + q_bytes, &ws)) return rc;
    w.s.row_ml = (float2*)ws;
    w.part = (float*)((char*)ws + ml_bytes);
    if (append)
        if (int rc = c.update(k_new, v_new, n_rows, stream)) return rc;
    if (t4)
        if (int rc = shared_turbo4_rotate_q(c, q, q_rows, w.s, stream)) return rc;
    if (int rc = launch_shared(nullptr, &c, w.s, stream)) return rc;
    if (int rc = launch_shared_merge(c.D, w.s, stream)) return rc;
    if (t4)
        if (int rc = launch_turbo4_rotate(c, w.s.out, (int)q_rows, true, (f16*)out, stream)) return rc;
    if (w.s.n_slots == 1) {
        hipLaunchKernelGGL(row_sums_kernel, dim3((R + 255) / 256, c.hkv), dim3(256), 0, stream, w.s);
        QW_HIP_CHECK(hipGetLastError());
    }
    if (q_bytes) {
        f16* const to = (f16*)((char*)ws + ml_bytes + part_bytes);
        const int64_t n = q_bytes / sizeof(f16);
        hipLaunchKernelGGL(copy_halves_kernel, dim3((unsigned)std::min<int64_t>((n + 255) / 256, 4096)), dim3(256), 0, stream,
                           (const f16*)q, to, n);
        QW_HIP_CHECK(hipGetLastError());
        w.s.q = to;
    }
    if (t4) return c.D == 256 ? launch_weights<4, 256, true>(w, stream) : launch_weights<4, 128, true>(w, stream);
    if (c.D == 256)
        return c.bits == 4   ? launch_weights<4, 256>(w, stream)
               : c.bits == 8 ? launch_weights<8, 256>(w, stream)
                             : launch_weights<16, 256>(w, stream);
    return c.bits == 4   ? launch_weights<4, 128>(w, stream)
           : c.bits == 8 ? launch_weights<8, 128>(w, stream)
                         : launch_weights<16, 128>(w, stream);
}

}  // namespace qw
