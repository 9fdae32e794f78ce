// evict.hip - eviction from a cache by accumulated key weights, gfx950.
//
// Per KV head h of a cache of T rows: keys t < sink and t >= T - recent stay, and of the
// others the budget - sink - recent of the largest weights[h][t]; equal weights go to the
// lower t, -0 equals 0, a NaN ranks below every number. The n = min(T, budget) kept rows move, code for
// code, in ascending order to rows 0 .. n - 1 of the destination (another cache, or the same one).
// Each head keeps its own set. The reference's caches shrink at the end only (KVCache::trim,
// crates/mlxcel-core/src/cache.rs:2251).
//
// The launches:
//   the select: the weight of the last kept key by its digits (11 + 11 + 10 bits of the float in
//     an order-preserving integer form, a histogram in LDS a digit), then the kept positions at the places that
//     scans of the counts before them give; a workgroup a head (evict_select_kernel) or, for
//     longer caches, one a chunk (evict_digit_kernel);
//   evict_rows_kernel copies 16-byte pieces: K rows whole; V, stored in 8-key blocks with the
//     8 keys of a dim together, key by key out of up to 8 source blocks.
// In place the rows go through a workspace: a row's new place may be another's old one.
// The select is bound by the latency of its dependent steps (32k keys of 4 heads 25 us in four launches), the
// copy by bandwidth: 48k of 64k fp16 rows, D = 256, 297 MB read (every line of V holds a kept
// key) and 197 written in 90 us, 5.5 TB/s; 16k of 131k 8-bit rows 151 MB in 32 us, 4.7 TB/s.
#include <algorithm>

#include "kv_cache.hpp"

namespace qw {

namespace {

constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64, kBins = 2048;
constexpr int kDigits = 3;
__host__ __device__ constexpr int digit_shift(int d) { return d == 0 ? 21 : d == 1 ? 10 : 0; }
__host__ __device__ constexpr int digit_bits(int d) { return d < 2 ? 11 : 10; }

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
    // the form of several workgroups a head (evict_digit_kernel): per head and chunk
    uint32_t* hist;                // [kDigits][hkv][chunks][kBins / 2]: two 16-bit counts a word
    uint32_t* above;               // [2][hkv][chunks]: keys above the cut by their first, second digit
    uint2* pick;                   // [kDigits][hkv]: the cut's digit, the kept keys left within it
    int chunks;
};

// Counts digit d of the KPT keys a thread holds as ranks into hist: those of the middle (bit e of mid)
// that share the cut's digits before it. Weights of 0, which keys that no row ever looked at have
// in common, would queue on one counter: a wave counts its own and adds them at once.
template <int KPT>
__device__ __forceinline__ void count_digit(uint32_t* hist, const uint32_t (&u)[KPT], uint32_t mid, int d, uint32_t prefix) {
    const int shift = digit_shift(d), bits = digit_bits(d);
    constexpr uint32_t kZero = 0x80000000u;  // the rank of 0
    uint32_t zeros = 0;
#pragma unroll
    for (int e = 0; e < KPT; e++) {
        const bool in = (mid >> e & 1) && (d == 0 || u[e] >> (shift + bits) == prefix);
        zeros += __popcll(__ballot(in && u[e] == kZero));
        if (in && u[e] != kZero) atomicAdd(&hist[u[e] >> shift & ((1u << bits) - 1)], 1u);
    }
    if (zeros && (threadIdx.x & 63) == 0) atomicAdd(&hist[kZero >> shift & ((1u << bits) - 1)], zeros);
}

// The sum of x over the threads before this one, over the workgroup; *total: over all.
__device__ __forceinline__ uint32_t scan_before(uint32_t x, uint32_t* s_wave, uint32_t* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t upto = x;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const uint32_t y = __shfl_up(upto, s);
        if (lane >= s) upto += y;
    }
    __syncthreads();  // s_wave is free
    if (lane == 63) s_wave[wave] = upto;
    __syncthreads();
    uint32_t before = upto - x, all = 0;
#pragma unroll
    for (int v = 0; v < kSelWaves; v++) {
        const uint32_t y = s_wave[v];
        before += v < wave ? y : 0u;
        all += y;
    }
    *total = all;
    return before;
}

// The bin in which the count from the top reaches left, and what is left within it: thread i
// holds the counts of bins kBins - 1 - 2 i (hi) and the one below it (lo).
__device__ __forceinline__ uint2 pick_bin(uint32_t hi, uint32_t lo, uint32_t left, uint32_t* s_wave, uint2* s_pick) {
    uint32_t total;
    const uint32_t before = scan_before(hi + lo, s_wave, &total);
    const int top = kBins - 1 - 2 * (int)threadIdx.x;
    if (left == 0 && threadIdx.x == 0) *s_pick = uint2{kBins - 1, 0u};  // (above every digit, or ties = 0)
    if (before < left && left <= before + hi)
        *s_pick = uint2{(uint32_t)top, left - before};
    else if (before + hi < left && left <= before + hi + lo)
        *s_pick = uint2{(uint32_t)top - 1, left - before - hi};
    __syncthreads();
    return *s_pick;
}

// Writes the kept keys among KPT consecutive ones a thread, from key t0: rank above the cut or
// outside the middle, and of those equal to it the first `ties` (eq0 of them and at0 kept keys in the
// chunks before). (A workgroup holds fewer than 2^16 keys: both counts in one scan.)
template <int KPT>
__device__ __forceinline__ void emit(const SelectArgs& a, int h, int t0, const float (&x)[KPT], const uint32_t (&u)[KPT],
                                     uint32_t mid, uint32_t cut, uint32_t ties, uint32_t at0, uint32_t eq0,
                                     uint32_t* s_wave) {
    uint32_t above = 0, equal = 0;  // bit e: key t0 + e
#pragma unroll
    for (int e = 0; e < KPT; e++) {
        const bool m = mid >> e & 1;
        above |= (uint32_t)(t0 + e < a.T && (!m || u[e] > cut)) << e;
        equal |= (uint32_t)(m && u[e] == cut) << e;
    }
    uint32_t total;
    const uint32_t before = scan_before((uint32_t)__popc(above) << 16 | (uint32_t)__popc(equal), s_wave, &total);
    uint32_t at = at0 + (before >> 16), eq = eq0 + (before & 0xFFFFu);
#pragma unroll
    for (int e = 0; e < KPT; e++) {
        const bool ab = above >> e & 1, eqe = equal >> e & 1;
        if (ab || (eqe && eq < ties)) {
            const uint32_t pos = at + min(eq, ties);
            a.kept[(int64_t)h * a.n + pos] = t0 + e;
            if (a.weights_out) a.weights_out[h * a.out_stride + pos] = x[e];
        }
        at += ab;
        eq += eqe;
    }
}

// The weights of a thread's keys; their ranks, and which of them lie in the middle.
template <int KPT>
__device__ __forceinline__ void load_keys(const SelectArgs& a, int h, int t0, float (&x)[KPT]) {
    const float* w = a.weights + h * a.stride;
#pragma unroll
    for (int e = 0; e < KPT; e++) x[e] = t0 + e < a.T ? w[t0 + e] : 0.0f;
}
template <int KPT>
__device__ __forceinline__ uint32_t rank_keys(const SelectArgs& a, int t0, const float (&x)[KPT], uint32_t (&u)[KPT]) {
    uint32_t mid = 0;
#pragma unroll
    for (int e = 0; e < KPT; e++) {
        u[e] = weight_rank(x[e]);
        mid |= (uint32_t)(t0 + e >= a.sink && t0 + e < a.T - a.recent) << e;
    }
    return mid;
}

// A head in one workgroup, its keys (KPT consecutive ones a thread) in registers.
template <int KPT>
__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(SelectArgs a) {
    __shared__ uint32_t hist[kBins];
    __shared__ uint32_t s_wave[kSelWaves];
    __shared__ uint2 s_pick;
    const int tid = threadIdx.x, h = blockIdx.x, t0 = tid * KPT;
    float x[KPT];
    uint32_t u[KPT];
    load_keys<KPT>(a, h, t0, x);
    const uint32_t mid = rank_keys<KPT>(a, t0, x, u);
    uint32_t prefix = 0, left = (uint32_t)a.need;
#pragma unroll
    for (int d = 0; d < kDigits; d++) {
        hist[2 * tid] = hist[2 * tid + 1] = 0;
        __syncthreads();
        count_digit<KPT>(hist, u, mid, d, prefix);
        __syncthreads();
        const uint2 p = pick_bin(hist[kBins - 1 - 2 * tid], hist[kBins - 2 - 2 * tid], left, s_wave, &s_pick);
        prefix = prefix << digit_bits(d) | (p.x & ((1u << digit_bits(d)) - 1));
        left = p.y;
    }
    emit<KPT>(a, h, t0, x, u, mid, prefix, left, 0, 0, s_wave);
}

// The same by chunks of kChunk keys, a workgroup each (grid (chunks, hkv)), in four launches: d = 0,
// 1, 2 count digit d of the chunk's keys that share the cut's digits before it (found from the last
// launch's counts by every workgroup for itself), d = 3 writes the kept keys.
constexpr int kChunkKeys = 4, kChunk = kSelThreads * kChunkKeys;

// f of a thread's word of the first n chunks' counts, 16 loads in flight.
template <class F>
__device__ __forceinline__ void for_chunks(const uint32_t* word, int n, F f) {
    for (int i = 0; i < n; i += 16) {
        uint32_t v[16];
#pragma unroll
        for (int j = 0; j < 16; j++) v[j] = word[(int64_t)min(i + j, n - 1) * (kBins / 2)];
#pragma unroll
        for (int j = 0; j < 16; j++) f(i + j < n ? v[j] : 0u);
    }
}

__global__ __launch_bounds__(kSelThreads) void evict_digit_kernel(SelectArgs a, int d) {
    __shared__ uint32_t hist[kBins];
    __shared__ uint32_t s_wave[kSelWaves];
    __shared__ uint2 s_pick;
    __shared__ uint32_t s_sum[2];
    const int tid = threadIdx.x, lane = tid & 63, c = blockIdx.x, h = blockIdx.y, hkv = gridDim.y;
    const int t0 = c * kChunk + tid * kChunkKeys;
    // (all loads first: the weights, the last digits picked, the last digit's counts)
    float x[kChunkKeys];
    uint32_t u[kChunkKeys];
    load_keys<kChunkKeys>(a, h, t0, x);
    hist[2 * tid] = hist[2 * tid + 1] = 0;
    if (tid < 2) s_sum[tid] = 0;
    const uint32_t* hist_d = nullptr;  // the last digit's counts of this head
    uint32_t prefix = 0, left = (uint32_t)a.need;
    if (d > 0) {
        hist_d = a.hist + ((int64_t)(d - 1) * hkv + h) * a.chunks * (kBins / 2);
        const uint2 p0 = a.pick[h], p1 = a.pick[hkv + h];  // (read where written: d > 1, d > 2)
        uint32_t n_hi = 0, n_lo = 0;
        for_chunks(hist_d + kBins / 2 - 1 - tid, a.chunks, [&](uint32_t v) {
            n_hi += v >> 16;
            n_lo += v & 0xFFFFu;
        });
        if (d > 1) prefix = p0.x, left = p0.y;
        if (d > 2) prefix = prefix << digit_bits(1) | p1.x, left = p1.y;
        const uint2 p = pick_bin(n_hi, n_lo, left, s_wave, &s_pick);
        if (c == 0 && tid == 0) a.pick[(d - 1) * hkv + h] = p;
        prefix = prefix << digit_bits(d - 1) | (p.x & ((1u << digit_bits(d - 1)) - 1));
        left = p.y;
    } else {
        __syncthreads();
    }
    const uint32_t mid = rank_keys<kChunkKeys>(a, t0, x, u);
    if (d < kDigits) {
        count_digit<kChunkKeys>(hist, u, mid, d, prefix);
        if (d > 0) {  // keys that the last digit put above the cut: the digits before it equal, it larger
            const int shift = digit_shift(d - 1), bits = digit_bits(d - 1);
            uint32_t n_above = 0;
#pragma unroll
            for (int e = 0; e < kChunkKeys; e++) {
                const uint32_t head = u[e] >> shift;
                n_above += __popcll(__ballot((mid >> e & 1) && head > prefix && (d == 1 || head >> bits == prefix >> bits)));
            }
            if (lane == 0 && n_above) atomicAdd(&s_sum[0], n_above);
        }
        __syncthreads();
        if (d > 0 && tid == 0) a.above[((d - 1) * hkv + h) * a.chunks + c] = s_sum[0];
        a.hist[(((int64_t)d * hkv + h) * a.chunks + c) * (kBins / 2) + tid] = hist[2 * tid] | hist[2 * tid + 1] << 16;
        return;
    }
    // kept keys above the cut and ties in the chunks before this one; protected ones too
    uint32_t n_above = 0, n_equal = 0;
    const uint32_t b2 = prefix & ((1u << digit_bits(2)) - 1);
    for_chunks(hist_d + tid, c, [&](uint32_t v) {
        n_above += (2u * tid > b2 ? v & 0xFFFFu : 0u) + (2u * tid + 1 > b2 ? v >> 16 : 0u);
        n_equal += (2u * tid == b2 ? v & 0xFFFFu : 0u) + (2u * tid + 1 == b2 ? v >> 16 : 0u);
    });
    for (int i = tid; i < c; i += kSelThreads)
        n_above += a.above[h * a.chunks + i] + a.above[(hkv + h) * a.chunks + i];
    if (n_above) atomicAdd(&s_sum[0], n_above);
    if (n_equal) atomicAdd(&s_sum[1], n_equal);
    __syncthreads();
    const int start = c * kChunk, lo = a.sink, hi = a.T - a.recent;
    const uint32_t at = s_sum[0] + min(start, lo) + max(0, start - hi);
    emit<kChunkKeys>(a, h, t0, x, u, mid, prefix, left, at, s_sum[1], s_wave);
}

// Keys up to which one workgroup a head does it. Four heads, one workgroup / chunks: 900 keys 5.9 / 19.5 us,
// 3500 8.8 / 20.7, 8000 19.0 / 24.0, 16000 25.0 / 24.8 (and three launches more); 32 keys a thread over 32000
// 52 / 25.
constexpr int kOneGroup = 16 * kSelThreads;

int launch_select(SelectArgs a, int hkv, int device, hipStream_t stream) {
    if (a.T <= kOneGroup) {
        auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(hkv), dim3(kSelThreads), 0, stream, a); };
        a.T <= kSelThreads ? run(evict_select_kernel<1>)
        : a.T <= 4 * kSelThreads ? run(evict_select_kernel<4>) : run(evict_select_kernel<16>);
        QW_HIP_CHECK(hipGetLastError());
        return QW_OK;
    }
    a.chunks = (a.T + kChunk - 1) / kChunk;
    const size_t per = (size_t)hkv * a.chunks;
    const size_t h_bytes = kDigits * per * (kBins / 2) * 4, p_bytes = kDigits * (size_t)hkv * sizeof(uint2);
    void* ws = nullptr;
    if (int rc = workspace(kWsSelect, device, stream, h_bytes + p_bytes + 2 * per * 4, &ws)) return rc;
    a.hist = (uint32_t*)ws;
    a.pick = (uint2*)((char*)ws + h_bytes);
    a.above = (uint32_t*)((char*)ws + h_bytes + p_bytes);
    for (int d = 0; d <= kDigits; d++) {
        hipLaunchKernelGGL(evict_digit_kernel, dim3(a.chunks, hkv), dim3(kSelThreads), 0, stream, a, d);
        QW_HIP_CHECK(hipGetLastError());
    }
    return QW_OK;
}

struct RowsCopy {
    const u32x4 *k, *v;      // source planes, as KvLayout has them
    const uint32_t *kp, *vp;
    u32x4 *k_to, *v_to;
    uint32_t *kp_to, *vp_to;
    const int32_t* kept;     // [hkv][n]
    const int* flag;         // the source's fast flag, copied where flag_to is not null
    int* flag_to;
    int n, n_out;            // kept rows; rows written, zeros from n on (a multiple of 8)
    int cap, cap_to, groups_v, kp_words;  // kp_words: words of a K row's params
    int row_major_v;         // Turbo4: V rows like K's, one params word a row
};

// BITS: of a code (or 16). Grid (groups, hkv), the first `groups_v` groups V's: a thread takes a
// 16-byte piece of V of a block's 8 rows, or of K (and of a row-major V) the same piece of each of
// the 8 rows. All its loads are issued before the first is used. Rows n .. n_out - 1 become zeros (V's
// codes in the last row's block that row's, under a scale and a bias of 0): what stands behind a
// cache's offset, up to the end of a tile, has weight 0 in its attention, and has to be finite.
template <int BITS, int D>
__global__ __launch_bounds__(256) void evict_rows_kernel(RowsCopy a) {
    constexpr int pieces = D * BITS / 16;  // of a block of V
    const int h = blockIdx.y, group = (int)blockIdx.x;
    const bool rows_of_v = a.row_major_v && group < a.groups_v;
    if (group >= a.groups_v || rows_of_v) {
        constexpr int ppr = pieces / 8;
        const uint32_t id = (uint32_t)(group - (rows_of_v ? 0 : a.groups_v)) * 256u + threadIdx.x;
        const int b = (int)(id / ppr), c = (int)(id % ppr);
        if (id == 0 && h == 0 && !rows_of_v && a.flag_to) *a.flag_to = *a.flag;
        if (8 * b >= a.n_out) return;
        const u32x4* from = rows_of_v ? a.v : a.k;
        u32x4* to = rows_of_v ? a.v_to : a.k_to;
        const uint32_t* pf = rows_of_v ? a.vp : a.kp;
        uint32_t* pt = rows_of_v ? a.vp_to : a.kp_to;
        const int32_t* kept = a.kept + (int64_t)h * a.n + 8 * b;
        const int rows = min(8, a.n - 8 * b), pw = a.row_major_v ? 1 : a.kp_words;
        const int64_t dst = (int64_t)h * a.cap_to + 8 * b;
        if (rows <= 0) {
#pragma unroll
            for (int k = 0; k < 8; k++) {
                to[(dst + k) * ppr + c] = u32x4{0, 0, 0, 0};
                if (c < pw) pt[(dst + k) * pw + c] = 0;
            }
            return;
        }
        int64_t src[8];
        u32x4 x[8];
        uint32_t p[8];
#pragma unroll
        for (int k = 0; k < 8; k++) src[k] = (int64_t)h * a.cap + kept[min(k, rows - 1)];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            x[k] = from[src[k] * ppr + c];
            p[k] = c < pw ? pf[src[k] * pw + c] : 0u;
        }
#pragma unroll
        for (int k = 0; k < 8; k++) {
            to[(dst + k) * ppr + c] = k < rows ? x[k] : u32x4{0, 0, 0, 0};
            if (c < pw) pt[(dst + k) * pw + c] = k < rows ? p[k] : 0u;
        }
        return;
    }
    const uint32_t id = (uint32_t)group * 256u + threadIdx.x;  // (past 2^31 from 67M fp16 rows of D = 256 on)
    const int pc = (int)(id % pieces);
    int b = (int)(id / pieces);
    if constexpr (pieces >= 64) b = __builtin_amdgcn_readfirstlane(b);  // a wave's pieces are one block's: its positions go through scalar loads
    if (8 * b >= a.n_out) return;
    const int32_t* kept = a.kept + (int64_t)h * a.n + 8 * b;
    const int rows = min(8, a.n - 8 * b);
    const int64_t sblk = (int64_t)h * (a.cap / 8), dblk = (int64_t)h * (a.cap_to / 8) + b;
    if (rows <= 0) {
        a.v_to[dblk * pieces + pc] = u32x4{0, 0, 0, 0};
        if (BITS != 16 && pc < a.kp_words * 2) ((u32x4*)a.vp_to)[dblk * a.kp_words * 2 + pc] = u32x4{0, 0, 0, 0};
        return;
    }
    int t[8];
#pragma unroll
    for (int k = 0; k < 8; k++) t[k] = kept[min(k, rows - 1)];
    // piece pc of the block: 4 dims' words of 8 nibbles, 2 dims' of 8 bytes or one dim's of 8
    // halves
    u32x4 out = {0, 0, 0, 0};
    if constexpr (BITS == 16) {
        uint32_t x[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            x[k] = ((const uint16_t*)(a.v + (sblk + t[k] / 8) * pieces + pc))[t[k] & 7];
            x[k] = k < rows ? x[k] : 0u;
        }
#pragma unroll
        for (int k = 0; k < 4; k++) out[k] = x[2 * k] | x[2 * k + 1] << 16;
    } else {
        u32x4 x[8];
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = a.v[(sblk + t[k] / 8) * pieces + pc];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int f = t[k] & 7;
            if constexpr (BITS == 4) {
                const int from = 4 * v4_nibble_pos(f), to = 4 * v4_nibble_pos(k);
#pragma unroll
                for (int j = 0; j < 4; j++) out[j] |= (x[k][j] >> from & 0xFu) << to;
            } else {
                const int from = 8 * (f & 3), to = 8 * (k & 3);
#pragma unroll
                for (int j = 0; j < 2; j++)
                    out[2 * j + k / 4] |= ((f & 4 ? x[k][2 * j + 1] : x[k][2 * j]) >> from & 0xFFu) << to;
            }
        }
    }
    a.v_to[dblk * pieces + pc] = out;
    if (BITS != 16 && pc < a.kp_words * 8) {  // scale and bias of key pc & 7 in group pc >> 3
        const int grp = pc >> 3, k = pc & 7;
        const int tk = kept[min(k, rows - 1)];
        const f16* from = (const f16*)a.vp + ((sblk + tk / 8) * a.kp_words + grp) * 16;
        f16* to = (f16*)a.vp_to + (dblk * a.kp_words + grp) * 16;
        const f16 scale = from[tk & 7], bias = from[8 + (tk & 7)];
        to[k] = k < rows ? scale : (f16)0.0f;
        to[8 + k] = k < rows ? bias : (f16)0.0f;
    }
}

// In place: the staged rows back to the cache's planes, in 16-byte pieces: grid (groups, hkv, plane).
struct BackCopy {
    const u32x4* from[4];
    u32x4* to[4];
    int64_t per_head[4], stride[4];  // pieces of a head's staged rows; of its rows in the cache
};
__global__ __launch_bounds__(256) void evict_back_kernel(BackCopy a) {
    const u32x4* from = a.from[0];
    u32x4* to = a.to[0];
    int64_t per = a.per_head[0], stride = a.stride[0];
#pragma unroll
    for (int p = 1; p < 4; p++)
        if ((int)blockIdx.z == p) from = a.from[p], to = a.to[p], per = a.per_head[p], stride = a.stride[p];
    const int h = blockIdx.y;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < per; i += (int64_t)gridDim.x * 256)
        to[h * stride + i] = from[h * per + i];
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
    // rows written: to a whole step of the capacity, which no tile of an attention kernel passes
    const int n_out = (int)(((int64_t)n + 255) / 256 * 256);
    const int64_t of_v = (int64_t)(n_out / 8) * (src.D * src.bits / 16), of_k = of_v / 8;  // threads of a head
    QW_REQUIRE(of_v + of_k + 512 <= UINT32_MAX, QW_ERR_UNSUPPORTED, "evict: too many rows for one call");
    DeviceGuard dg(src.device);
    QW_REQUIRE(dg.ok, QW_ERR_HIP, "evict: hipSetDevice failed");
    if (dst.cap < n) {
        hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
        QW_HIP_CHECK(hipStreamIsCapturing(stream, &cs));
        QW_REQUIRE(cs == hipStreamCaptureStatusNone, QW_ERR_STATE,
                   "evict: the destination has to grow and the stream is being captured; reserve it before");
        if (int rc = dst.reserve(n, stream)) return rc;
    }
    // in place the rows that move are staged: planes of n_out rows a head
    char* ws = nullptr;
    size_t at[4] = {0, src.k_data_bytes(n_out), 0, 0};
    at[2] = at[1] + src.v_data_bytes(n_out);
    at[3] = at[2] + src.k_param_bytes(n_out);
    const bool staged = in_place && n < T;
    if (staged) {
        void* p = nullptr;
        if (int rc = workspace(kWsEvict, src.device, stream, at[3] + src.v_param_bytes(n_out), &p)) return rc;
        ws = (char*)p;
    }
    const int first = std::min(sink, T), last = std::min(recent, T - first);  // (first + last <= n)
    SelectArgs s{weights, weights_stride, T, n, first, last, n - first - last, kept, weights_out, weights_out_stride};
    if (int rc = launch_select(s, src.hkv, src.device, stream)) return rc;
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
    c.n = n;
    c.n_out = n_out;
    c.cap = src.cap;
    c.cap_to = staged ? n_out : dst.cap;
    c.kp_words = src.affine() ? src.D / kGroup : src.turbo4() ? 1 : 0;
    c.row_major_v = src.turbo4() ? 1 : 0;
    c.groups_v = (int)((src.turbo4() ? of_k + 255 : of_v + 255) / 256);
    const dim3 grid((unsigned)(c.groups_v + (of_k + 255) / 256), src.hkv);
    auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, c); };
    if (src.D == 256)
        src.bits == 4 ? launch(evict_rows_kernel<4, 256>) : src.bits == 8 ? launch(evict_rows_kernel<8, 256>) : launch(evict_rows_kernel<16, 256>);
    else
        src.bits == 4 ? launch(evict_rows_kernel<4, 128>) : src.bits == 8 ? launch(evict_rows_kernel<8, 128>) : launch(evict_rows_kernel<16, 128>);
    QW_HIP_CHECK(hipGetLastError());
    if (staged) {
        void* const to[4] = {src.k_data, src.v_data, src.k_params, src.v_params};
        const size_t per[4] = {src.k_data_bytes(n_out), src.v_data_bytes(n_out), src.k_param_bytes(n_out),
                               src.v_param_bytes(n_out)};
        const size_t full[4] = {src.k_data_bytes(src.cap), src.v_data_bytes(src.cap), src.k_param_bytes(src.cap),
                                src.v_param_bytes(src.cap)};
        BackCopy b;
        for (int i = 0; i < 4; i++) {
            b.from[i] = (const u32x4*)(ws + at[i]);
            b.to[i] = (u32x4*)to[i];
            b.per_head[i] = per[i] / src.hkv / 16;
            b.stride[i] = full[i] / src.hkv / 16;
        }
        const int64_t groups = std::min<int64_t>((b.per_head[0] + 255) / 256, 1024);
        hipLaunchKernelGGL(evict_back_kernel, dim3((unsigned)groups, src.hkv, src.bits == 16 ? 2 : 4), dim3(256), 0, stream, b);
        QW_HIP_CHECK(hipGetLastError());
    }
    dst.offset = n;
    return QW_OK;
}

}  // namespace qw
