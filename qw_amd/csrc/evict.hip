// evict.hip - eviction from a cache by accumulated key weights, gfx950.
//
// Per KV head h of a cache of T rows: keys t < sink and t >= T - recent stay, and of the
// others the budget - sink - recent of the largest weights[h][t]; equal weights go to the
// lower t, -0 equals 0, a NaN ranks below every number. The n = min(T, budget) kept rows move, code for
// code, in ascending order to rows 0 .. n - 1 of the destination (another cache, or the same one).
// Each head keeps its own set. The reference's caches shrink at the end only (KVCache::trim,
// crates/mlxcel-core/src/cache.rs:2251).
//
// Two launches (three in place):
//   evict_select_kernel, a workgroup a head: a radix select finds the weight of the last kept
//     key (11 + 11 + 10 bits of the float in an order-preserving integer form, one LDS histogram a digit),
//     then each wave walks a run of the keys and writes the kept positions at the places that
//     counts of the runs before it give;
//   evict_rows_kernel copies 16-byte pieces: K rows whole; V, stored in 8-key blocks with the
//     8 keys of a dim together, key by key out of up to 8 source blocks.
// In place the rows go through a workspace: a row's new place may be another's old one.
#include <algorithm>

#include "kv_cache.hpp"

namespace qw {

namespace {

constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64, kBins = 2048;

// Order-preserving: larger weight, larger integer; NaN 0.
__device__ __forceinline__ uint32_t weight_rank(float w) {
    const uint32_t u = __float_as_uint(w == 0.0f ? 0.0f : w);
    if (w != w) return 0u;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct SelectArgs {
    const float* weights;
    int64_t stride;
    int T, n, sink, recent, need;  // need: kept keys of the middle [sink, T - recent)
    int32_t* kept;                 // [hkv][n]
    float* weights_out;            // [hkv][out_stride] or null
    int64_t out_stride;
};

__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(SelectArgs a) {
    __shared__ uint32_t hist[kBins];
    __shared__ uint32_t s_wave[kSelWaves][2];
    __shared__ uint32_t s_pick[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = blockIdx.x;
    const float* w = a.weights + h * a.stride;
    const int lo = a.sink, hi = a.T - a.recent;  // the middle
    // the rank of the last kept key, digit by digit; left: kept keys among those that share
    // the digits so far
    uint32_t prefix = 0, left = (uint32_t)a.need;
    const int shifts[3] = {21, 10, 0};
    for (int d = 0; d < 3; d++) {
        const int shift = shifts[d], bits = d < 2 ? 11 : 10;
        for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
        __syncthreads();
        for (int t = lo + tid; t < hi; t += kSelThreads) {
            const uint32_t u = weight_rank(w[t]);
            const bool in = d == 0 || (u >> (shift + bits)) == prefix;
            const uint32_t bin = (u >> shift) & ((1u << bits) - 1);
            if (in) atomicAdd(&hist[bin], 1u);
        }
        __syncthreads();
        // the bin in which the count from the top reaches left
        if (wave == 0) {
            uint32_t mine = 0;
            for (int i = 0; i < kBins / 64; i++) mine += hist[kBins - 1 - (lane * (kBins / 64) + i)];
            uint32_t upto = mine;
            for (int s = 1; s < 64; s <<= 1) {
                const uint32_t x = __shfl_up(upto, s);
                if (lane >= s) upto += x;
            }
            const uint32_t before = upto - mine;
            if (before < left && left <= upto) {
                uint32_t c = before;
                for (int i = 0; i < kBins / 64; i++) {
                    const int b = kBins - 1 - (lane * (kBins / 64) + i);
                    if (c + hist[b] >= left) {
                        s_pick[0] = b;
                        s_pick[1] = left - c;
                        break;
                    }
                    c += hist[b];
                }
            }
            if (left == 0 && lane == 0) s_pick[0] = (1u << bits) - 1, s_pick[1] = 0;
        }
        __syncthreads();
        prefix = prefix << bits | s_pick[0];
        left = s_pick[1];
        __syncthreads();
    }
    const uint32_t cut = prefix, ties = left;  // kept: rank > cut, and the first `ties` of rank == cut
    // need == 0: nothing above the largest integer, no ties
    // runs of whole 64-key steps a wave
    const int per = ((a.T + kSelWaves - 1) / kSelWaves + 63) / 64 * 64;
    const int r0 = min(a.T, wave * per), r1 = min(a.T, r0 + per);
    uint32_t above = 0, equal = 0;
    for (int t = r0 + lane; t < r1; t += 64) {
        const bool mid = t >= lo && t < hi;
        const uint32_t u = mid ? weight_rank(w[t]) : 0;
        above += !mid || u > cut;
        equal += mid && u == cut;
    }
    for (int s = 32; s; s >>= 1) {
        above += __shfl_xor(above, s);
        equal += __shfl_xor(equal, s);
    }
    if (lane == 0) {
        s_wave[wave][0] = above;
        s_wave[wave][1] = equal;
    }
    __syncthreads();
    uint32_t at = 0, eq = 0;  // kept keys above the cut and ties in the runs before this one
    for (int v = 0; v < wave; v++) {
        at += s_wave[v][0];
        eq += s_wave[v][1];
    }
    int32_t* kept = a.kept + (int64_t)h * a.n;
    for (int t = r0 + lane; t - lane < r1; t += 64) {
        const bool in = t < r1, mid = t >= lo && t < hi;
        const float x = in ? w[t] : 0.0f;
        const uint32_t u = weight_rank(x);
        const uint64_t m_above = __ballot(in && (!mid || u > cut)), m_equal = __ballot(in && mid && u == cut);
        const uint64_t below = ((uint64_t)1 << lane) - 1;
        const uint32_t tie = eq + __popcll(m_equal & below);  // ties before this key
        const bool keep = (m_above >> lane & 1) || ((m_equal >> lane & 1) && tie < ties);
        const uint32_t pos = at + __popcll(m_above & below) + min(tie, ties);
        if (keep) {
            kept[pos] = t;
            if (a.weights_out) a.weights_out[h * a.out_stride + pos] = x;
        }
        at += __popcll(m_above);
        eq += __popcll(m_equal);
    }
}

struct RowsCopy {
    const u32x4 *k, *v;      // source planes, as KvLayout has them
    const uint32_t *kp, *vp;
    u32x4 *k_to, *v_to;
    uint32_t *kp_to, *vp_to;
    const int32_t* kept;     // [hkv][n]
    const int* flag;         // the source's fast flag, copied where flag_to is not null
    int* flag_to;
    int hkv, n, cap, cap_to, bits, D, kp_words;  // kp_words: words of a K row's params
    int row_major_v;         // Turbo4: V rows like K's, one params word a row
};

// BITS: of a code (or 16). A thread copies one 16-byte piece of one 8-row block of one plane.
template <int BITS>
__global__ __launch_bounds__(256) void evict_rows_kernel(RowsCopy a) {
    const int pieces = a.D * BITS / 16;  // of a block, in each plane
    const int64_t n_blk = (a.n + 7) / 8, total = a.hkv * n_blk * 2 * pieces;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id == 0 && a.flag_to) *a.flag_to = *a.flag;
    if (id >= total) return;
    const int pc = (int)(id % pieces), plane = (int)(id / pieces % 2);
    const int64_t hb = id / pieces / 2;
    const int h = (int)(hb / n_blk), b = (int)(hb % n_blk);
    const int32_t* kept = a.kept + (int64_t)h * a.n + 8 * b;
    const int rows = min(8, a.n - 8 * b);
    if (plane == 0 || a.row_major_v) {
        const u32x4* from = plane == 0 ? a.k : a.v;
        u32x4* to = plane == 0 ? a.k_to : a.v_to;
        const int ppr = pieces / 8, r = pc / ppr, c = pc % ppr;
        if (r >= rows) return;
        const int64_t src = (int64_t)h * a.cap + kept[r], dst = (int64_t)h * a.cap_to + 8 * b + r;
        to[dst * ppr + c] = from[src * ppr + c];
        const uint32_t* pf = plane == 0 ? a.kp : a.vp;
        uint32_t* pt = plane == 0 ? a.kp_to : a.vp_to;
        const int pw = a.row_major_v ? 1 : a.kp_words;
        if (c < pw) pt[dst * pw + c] = pf[src * pw + c];
        return;
    }
    const int64_t sblk = (int64_t)h * (a.cap / 8), dblk = (int64_t)h * (a.cap_to / 8) + b;
    // piece pc of the block: 4 dims' words of 8 nibbles, 2 dims' of 8 bytes or one dim's of 8 halves
    u32x4 out = {0, 0, 0, 0}, x = {0, 0, 0, 0};
    int have = -1;
#pragma unroll
    for (int k = 0; k < 8; k++) {
        if (k >= rows) break;
        const int t = kept[k];
        if (t / 8 != have) {
            have = t / 8;
            x = a.v[(sblk + have) * pieces + pc];
        }
        const int f = t & 7;
        if constexpr (BITS == 4) {
            const int from = 4 * v4_nibble_pos(f), to = 4 * v4_nibble_pos(k);
#pragma unroll
            for (int j = 0; j < 4; j++) out[j] |= (x[j] >> from & 0xFu) << to;
        } else if constexpr (BITS == 8) {
            const int from = 8 * (f & 3), to = 8 * (k & 3);
#pragma unroll
            for (int j = 0; j < 2; j++) out[2 * j + k / 4] |= ((f & 4 ? x[2 * j + 1] : x[2 * j]) >> from & 0xFFu) << to;
        } else {
            const uint32_t w = f & 4 ? (f & 2 ? x[3] : x[2]) : (f & 2 ? x[1] : x[0]);
            out[k / 2] |= (w >> (16 * (f & 1)) & 0xFFFFu) << (16 * (k & 1));
        }
    }
    a.v_to[dblk * pieces + pc] = out;
    if (BITS != 16 && pc < a.kp_words * 8) {  // scale and bias of key pc & 7 in group pc >> 3
        const int grp = pc >> 3, k = pc & 7;
        if (k < rows) {
            const int t = kept[k];
            const f16* from = (const f16*)a.vp + ((sblk + t / 8) * a.kp_words + grp) * 16;
            f16* to = (f16*)a.vp_to + (dblk * a.kp_words + grp) * 16;
            to[k] = from[t & 7];
            to[8 + k] = from[8 + (t & 7)];
        }
    }
}

// In place: the staged rows (cap_to rows a head) back to the cache's planes; 16-byte pieces.
__global__ __launch_bounds__(256) void evict_back_kernel(const u32x4* __restrict__ from, u32x4* __restrict__ to,
                                                         int64_t per_head, int64_t from_stride, int64_t to_stride,
                                                         int64_t total) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t h = i / per_head, r = i % per_head;
        to[h * to_stride + r] = from[h * from_stride + r];
    }
}

}  // namespace

int evict(KVCache& src, KVCache* into, const float* weights, int64_t weights_stride, int budget, int sink, int recent,
          int32_t* kept, float* weights_out, int64_t weights_out_stride, int* n_kept, hipStream_t stream) {
    KVCache& dst = into ? *into : src;
    const bool in_place = &dst == &src;
    QW_REQUIRE(src.offset == 0 || (weights && kept), QW_ERR_INVALID_ARGUMENT, "evict: null weights/kept");
    QW_REQUIRE(budget > 0 && sink >= 0 && recent >= 0 && (int64_t)sink + recent <= budget, QW_ERR_INVALID_ARGUMENT,
               "evict: budget > 0 and sink + recent <= budget, neither negative");
    QW_REQUIRE(dst.mode == src.mode && dst.hkv == src.hkv && dst.D == src.D && dst.device == src.device &&
                   (!src.turbo4() || dst.turbo_seed == src.turbo_seed),
               QW_ERR_INVALID_ARGUMENT, "evict: the destination needs the cache's mode, heads, head_dim, seed and device");
    const int T = src.offset, n = std::min(T, budget);
    QW_REQUIRE(weights_stride >= T && (!weights_out || weights_out_stride >= n), QW_ERR_INVALID_ARGUMENT,
               "evict: a weights stride below its row's length");
    if (weights_out && T > 0) {
        const uintptr_t a0 = (uintptr_t)weights, a1 = a0 + 4 * ((uint64_t)(src.hkv - 1) * weights_stride + T);
        const uintptr_t b0 = (uintptr_t)weights_out, b1 = b0 + 4 * ((uint64_t)(src.hkv - 1) * weights_out_stride + n);
        QW_REQUIRE(a1 <= b0 || b1 <= a0, QW_ERR_INVALID_ARGUMENT, "evict: weights_out overlaps weights");
    }
    if (n_kept) *n_kept = n;
    if (T == 0) {
        dst.offset = 0;
        return QW_OK;
    }
    DeviceGuard dg(src.device);
    QW_REQUIRE(dg.ok, QW_ERR_HIP, "evict: hipSetDevice failed");
    if (dst.cap < n) {
        hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
        QW_HIP_CHECK(hipStreamIsCapturing(stream, &cs));
        QW_REQUIRE(cs == hipStreamCaptureStatusNone, QW_ERR_STATE,
                   "evict: the destination has to grow and the stream is being captured; reserve it before");
        if (int rc = dst.reserve(n, stream)) return rc;
    }
    // in place the rows that move are staged: planes of n rows a head, in whole 8-row blocks
    const int rows8 = (n + 7) / 8 * 8;
    char* ws = nullptr;
    size_t at[4] = {0, src.k_data_bytes(rows8), 0, 0};
    at[2] = at[1] + src.v_data_bytes(rows8);
    at[3] = at[2] + (src.k_param_bytes(rows8) + 15) / 16 * 16;
    const bool staged = in_place && n < T;
    if (staged) {
        void* p = nullptr;
        if (int rc = workspace(kWsEvict, src.device, stream, at[3] + src.v_param_bytes(rows8), &p)) return rc;
        ws = (char*)p;
    }
    const int first_need = std::max(0, n - std::min(sink, T) - std::min(recent, T - std::min(sink, T)));
    SelectArgs s{weights, weights_stride, T, n, std::min(sink, T), std::min(recent, T - std::min(sink, T)), first_need,
                 kept, weights_out, weights_out_stride};
    hipLaunchKernelGGL(evict_select_kernel, dim3(src.hkv), dim3(kSelThreads), 0, stream, s);
    QW_HIP_CHECK(hipGetLastError());
    if (in_place && n == T) return QW_OK;  // every row stays where it is
    RowsCopy c{};
    c.k = (const u32x4*)src.k_data;
    c.v = (const u32x4*)src.v_data;
    c.kp = src.k_params;
    c.vp = src.v_params;
    c.k_to = (u32x4*)(staged ? ws : (char*)dst.k_data);
    c.v_to = (u32x4*)(staged ? ws + at[1] : (char*)dst.v_data);
    c.kp_to = (uint32_t*)(staged ? ws + at[2] : (char*)dst.k_params);
    c.vp_to = (uint32_t*)(staged ? ws + at[3] : (char*)dst.v_params);
    c.kept = kept;
    c.flag = src.fast_flag;
    c.flag_to = in_place ? nullptr : dst.fast_flag;
    c.hkv = src.hkv;
    c.n = n;
    c.cap = src.cap;
    c.cap_to = staged ? rows8 : dst.cap;
    c.bits = src.bits;
    c.D = src.D;
    c.kp_words = src.affine() ? src.D / kGroup : src.turbo4() ? 1 : 0;
    c.row_major_v = src.turbo4() ? 1 : 0;
    const int64_t pieces = (int64_t)src.hkv * (rows8 / 8) * 2 * (src.D * src.bits / 16);
    const dim3 grid((unsigned)((pieces + 255) / 256));
    if (src.bits == 4)
        hipLaunchKernelGGL(evict_rows_kernel<4>, grid, dim3(256), 0, stream, c);
    else if (src.bits == 8)
        hipLaunchKernelGGL(evict_rows_kernel<8>, grid, dim3(256), 0, stream, c);
    else
        hipLaunchKernelGGL(evict_rows_kernel<16>, grid, dim3(256), 0, stream, c);
    QW_HIP_CHECK(hipGetLastError());
    if (staged) {
        void* const to[4] = {src.k_data, src.v_data, src.k_params, src.v_params};
        const size_t per[4] = {src.k_data_bytes(rows8), src.v_data_bytes(rows8), src.k_param_bytes(rows8),
                               src.v_param_bytes(rows8)};
        const size_t full[4] = {src.k_data_bytes(src.cap), src.v_data_bytes(src.cap), src.k_param_bytes(src.cap),
                                src.v_param_bytes(src.cap)};
        for (int i = 0; i < 4; i++) {
            if (!per[i]) continue;
            const int64_t ph = per[i] / src.hkv / 16, total = ph * src.hkv;
            hipLaunchKernelGGL(evict_back_kernel, dim3((unsigned)std::min<int64_t>((total + 255) / 256, 2048)),
                               dim3(256), 0, stream, (const u32x4*)(ws + at[i]), (u32x4*)to[i], ph, ph,
                               (int64_t)(full[i] / src.hkv / 16), total);
            QW_HIP_CHECK(hipGetLastError());
        }
    }
    dst.offset = n;
    return QW_OK;
}

}  // namespace qw
