// paged_select.hip - which pages of a sequence each KV head reads for its newest tokens.
//
// No key of a page scores more than sum_d max(q_d hi_d, q_d lo_d), with hi and lo the page's largest and
// least key of each dim. The bounds are kept as 8-bit codes over the page's largest magnitude (paged.hpp),
// q becomes 8-bit codes over its rows' largest magnitude, and the sum is of whole numbers:
//   score(page) = top(page) * max over rows of sum_d (max(q_d, 0) hi_d + min(q_d, 0) lo_d)
// with one rounding, so that the picks do not depend on any order of summation. It is a product of
// matrices of 2 D codes (v_mfma_i32_16x16x64_i8: 16 pages by 16 rows), bound by reading 2 D + 4 bytes a page (32 sequences
// of 1024 pages, 8 KV heads, D = 128: 68 MB in 14.3 us, 4.8 TB/s).
// A second launch finds the score of the last page that stays: a histogram of the scores in LDS gives its bin, the
// bin's few members are ranked one against the other (where they are many, as with ties, the score is found two
// bits a step over the keys, which wait in registers), and the picks are written in ascending order.
#include <algorithm>

#include "paged.hpp"

namespace qw {

namespace {

typedef int int4v __attribute__((ext_vector_type(4)));

constexpr int kMaxPages = 65536;

struct SelectArgs {
    PagedView c;
    const f16* q;
    int64_t q_seq, q_head, q_row;
    const int32_t* lengths;
    const int32_t* table;
    int64_t table_stride;
    int width, G, n_rows, R;
    int budget, sink, recent;
    int tiles;      // tiles of 16 pages a wave
    float* scores;  // [n_seq][hkv][width]
    int32_t* picked;  // [n_seq][hkv][budget]
};

__device__ __forceinline__ int pages_of(const SelectArgs& a, int b) {
    const int len = min(max(a.lengths[b], 0), a.width << a.c.lg);
    return (len + (1 << a.c.lg) - 1) >> a.c.lg;
}

template <int CTRL>
__device__ __forceinline__ int dpp_max(int x) {
    return max(x, __builtin_amdgcn_update_dpp(x, x, CTRL, 0xF, 0xF, false));
}

template <int D>
__global__ __launch_bounds__(256) void paged_score_kernel(SelectArgs a) {
    constexpr int STEPS = D / 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
    const int h = blockIdx.y, b = blockIdx.z;
    const int first = ((int)blockIdx.x * 4 + wave) * a.tiles * 16;
    if (first >= a.width) return;  // (no barrier follows)
    // the bounds of 16 pages: requested before the queries' codes form
    struct Bounds {
        int4v x[2 * STEPS];
        float top;
        bool there;
    } cur, next;
    auto page_at = [&](int p0) { return a.table[b * a.table_stride + min(p0 + col, a.width - 1)]; };
    auto load = [&](Bounds& to, int page) {
        to.there = (uint32_t)page < (uint32_t)a.c.n_pages;
        const int64_t ph = (int64_t)(to.there ? page : 0) * a.c.hkv + h;
        const int8_t* codes = a.c.codes + ph * 2 * D + 16 * g;
        to.top = a.c.top[ph];
#pragma unroll
        for (int j = 0; j < 2 * STEPS; j++) to.x[j] = *(const int4v*)(codes + 64 * j);
    };
    const int page0 = page_at(first), page1 = page_at(first + 16);
    load(cur, page0);
    const int pages = pages_of(a, b);
    if (pages <= a.budget || first >= pages) return;  // (they all stay)
    auto row_at = [&](int tile) {
        const int row = min(16 * tile + col, a.R - 1);
        return a.q + b * a.q_seq + (int64_t)(h * a.G + row / a.n_rows) * a.q_head + row % a.n_rows * a.q_row + 16 * g;
    };
    const int row_tiles = (a.R + 15) / 16;
    float big = 0.0f;
    for (int t = 0; t < row_tiles; t++) {
        const f16* q = row_at(t);
#pragma unroll
        for (int j = 0; j < STEPS; j++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const half8 x = *(const half8*)(q + 64 * j + 8 * e);
#pragma unroll
                for (int i = 0; i < 8; i++) big = fmaxf(big, fabsf((float)x[i]));
            }
    }
    big = wave_reduce(big, [](float x, float y) { return fmaxf(x, y); });
    const float inv = big > 0.0f ? 127.0f / big : 0.0f;
    const int last = min(first + a.tiles * 16, pages);
    float* scores = a.scores + ((int64_t)b * a.c.hkv + h) * a.width;
    for (int t = 0; t < row_tiles; t++) {
        const f16* q = row_at(t);
        int4v up[STEPS], down[STEPS];
#pragma unroll
        for (int j = 0; j < STEPS; j++)
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const half4v x = *(const half4v*)(q + 64 * j + 4 * w);
                uint32_t u = 0, d = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int c = (int)fminf(fmaxf(__builtin_rintf((float)x[i] * inv), -127.0f), 127.0f);
                    u |= (uint32_t)max(c, 0) << (8 * i);
                    d |= ((uint32_t)min(c, 0) & 0xFFu) << (8 * i);
                }
                up[j][w] = (int)u, down[j][w] = (int)d;
            }
        const bool real = 16 * t + col < a.R;
        if (t > 0) load(cur, page0);
        int ahead = page1;  // the page behind the next 16's bounds, which are on their way
        for (int p0 = first; p0 < last; p0 += 16) {
            if (p0 + 16 < last) {
                load(next, ahead);
                ahead = page_at(p0 + 32);
            }
            int4v acc = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < STEPS; j++) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(cur.x[j], up[j], acc, 0, 0, 0);
#pragma unroll
            for (int j = 0; j < STEPS; j++) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(cur.x[STEPS + j], down[j], acc, 0, 0, 0);
            // pages p0 + 4 g + i: the largest of the 16 rows
            int best[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                int m = real ? acc[i] : INT32_MIN;
                m = dpp_max<0xB1>(m);
                m = dpp_max<0x4E>(m);
                m = dpp_max<0x124>(m);
                best[i] = dpp_max<0x128>(m);
            }
            // lane col writes page p0 + col: its rows' largest lie in lanes 16 (col / 4) ..
            const int from = 16 * (col >> 2);
            const int b0 = __shfl(best[0], from), b1 = __shfl(best[1], from), b2 = __shfl(best[2], from), b3 = __shfl(best[3], from);
            const int m = col & 2 ? (col & 1 ? b3 : b2) : (col & 1 ? b1 : b0);
            if (g == 0 && p0 + col < last) {
                float s = cur.there ? cur.top * (float)m + 0.0f : -INFINITY;  // (-0 becomes 0)
                if (t > 0) s = fmaxf(s, scores[p0 + col]);
                scores[p0 + col] = s;
            }
            cur = next;
        }
    }
}

__device__ __forceinline__ uint32_t wave_sum(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(x), 63);
}

// Whole numbers that order as the scores do; 0 for none.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float unordered(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}
constexpr uint32_t kNoPage = 0x007FFFFFu;  // ordered(-infinity): a column that names no page
constexpr int kBins = 2048, kMembers = 256;

// KPT scores a thread in registers, or (0) as many as there are, read again where they are looked at.
template <int NT, int KPT>
__global__ __launch_bounds__(NT) void paged_pick_kernel(SelectArgs a) {
    constexpr int NW = NT / 64;
    __shared__ uint32_t sm[2][NW][4], hist[kBins], found[4];
    __shared__ uint2 member[kMembers];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int h = blockIdx.x, b = blockIdx.y;
    const float* scores = a.scores + ((int64_t)b * a.c.hkv + h) * a.width;
    const int per_thread = KPT ? KPT : (a.width + NT - 1) / NT;
    const int first = wave * 64 * per_thread + lane;
    constexpr int U = KPT ? KPT : 1;
    float score[U];
    if constexpr (KPT > 0) {  // (with the lengths; what stands behind a sequence's pages is not looked at)
#pragma unroll
        for (int i = 0; i < KPT; i++) score[i] = a.width > a.budget && first + 64 * i < a.width ? scores[first + 64 * i] : 0.0f;
    }
    const int n = pages_of(a, b);
    int32_t* picked = a.picked + ((int64_t)b * a.c.hkv + h) * a.budget;
    if (n <= a.budget) {
        for (int i = threadIdx.x; i < a.budget; i += NT) picked[i] = i < n ? i : -1;
        return;
    }
    const int lo = a.sink, hi = n - a.recent;
    const uint32_t need = (uint32_t)(a.budget - a.sink - a.recent);
    uint32_t key[U];
    if constexpr (KPT > 0) {
#pragma unroll
        for (int i = 0; i < KPT; i++) {
            const int p = first + 64 * i;
            key[i] = p >= lo && p < hi ? ordered(score[i]) : 0u;
        }
    }
    auto key_at = [&](int i) {
        if constexpr (KPT > 0) return key[i];
        const int p = first + 64 * i;
        return p >= lo && p < hi ? ordered(scores[p]) : 0u;
    };
    float least_f = INFINITY, most_f = -INFINITY;  // of the scores of pages that there are
#pragma unroll U
    for (int i = 0; i < per_thread; i++) {
        const uint32_t k = key_at(i);
        if (k > kNoPage) least_f = OpMin()(least_f, unordered(k)), most_f = OpMax()(most_f, unordered(k));
    }
    least_f = wave_reduce(least_f, OpMin());
    most_f = wave_reduce(most_f, OpMax());
    if (lane == 0) sm[0][wave][0] = __float_as_uint(least_f), sm[0][wave][1] = __float_as_uint(most_f);
    for (int i = threadIdx.x; i < kBins; i += NT) hist[i] = 0;
    if (threadIdx.x == 0) found[2] = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; w++) {
        least_f = OpMin()(least_f, __uint_as_float(sm[0][w][0]));
        most_f = OpMax()(most_f, __uint_as_float(sm[0][w][1]));
    }
    uint32_t cut = ~0u;
    bool few = true;
    if (need > 0) {
        // bins grow with the scores (differences, products and whole parts keep an order), the lowest for what has none
        const float per = (float)kBins / (most_f - least_f);
        auto bin_of = [&](uint32_t k) { return (int)fminf(fmaxf((unordered(k) - least_f) * per, 0.0f), (float)(kBins - 1)); };
#pragma unroll U
        for (int i = 0; i < per_thread; i++) {
            const uint32_t k = key_at(i);
            if (k) atomicAdd(&hist[bin_of(k)], 1u);
        }
        __syncthreads();
        // the bin in which the sum from the top reaches `need`
        constexpr int PER = kBins / NT;
        uint32_t mine[PER], sum = 0;
#pragma unroll
        for (int i = 0; i < PER; i++) sum += mine[i] = hist[kBins - 1 - ((int)threadIdx.x * PER + i)];
        uint32_t through = wave_scan(sum);
        if (lane == 63) sm[1][wave][0] = through;
        __syncthreads();
        for (int w = 0; w < wave; w++) through += sm[1][w][0];
        if (through >= need && through - sum < need) {
            uint32_t above = through - sum;
            int i = 0;
#pragma unroll
            for (int k = 0; k < PER - 1; k++)
                if (i == k && above + mine[k] < need) above += mine[k], i++;
            found[0] = kBins - 1 - (threadIdx.x * PER + i);
            found[1] = above;
            found[3] = hist[kBins - 1 - (threadIdx.x * PER + i)];
        }
        __syncthreads();
        const int bin = (int)found[0];
        few = found[3] <= kMembers;
        if (few) {
#pragma unroll U
            for (int i = 0; i < per_thread; i++) {
                const uint32_t k = key_at(i);
                if (k && bin_of(k) == bin) member[atomicAdd(&found[2], 1u)] = uint2{k, (uint32_t)(first + 64 * i)};
            }
            __syncthreads();
            const uint32_t members = found[3], room = need - found[1];
            if (threadIdx.x < members) {
                const uint2 me = member[threadIdx.x];
                uint32_t before = 0;
                for (uint32_t i = 0; i < members; i++) {
                    const uint2 x = member[i];
                    before += x.x > me.x || (x.x == me.x && x.y < me.y);
                }
                if (before + 1 == room) found[0] = me.x;
            }
            __syncthreads();
            cut = __builtin_amdgcn_readfirstlane(found[0]);
        }
    }
    // many members: the largest value that `need` keys reach; bits above the highest that differs are common to all
    if (!few) {
        uint32_t least = ~0u, most = 0;
#pragma unroll U
        for (int i = 0; i < per_thread; i++) {
            const uint32_t k = key_at(i);
            if (k) least = min(least, k), most = max(most, k);
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            least = min(least, (uint32_t)__shfl_xor((int)least, d));
            most = max(most, (uint32_t)__shfl_xor((int)most, d));
        }
        if (lane == 0) sm[0][wave][0] = least, sm[0][wave][1] = most;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NW; w++) least = min(least, sm[0][w][0]), most = max(most, sm[0][w][1]);
        least = __builtin_amdgcn_readfirstlane(least);
        most = __builtin_amdgcn_readfirstlane(most);
        const int top = least == most ? 0 : 32 - __builtin_clz(least ^ most);  // bits to find
        int shift = (top + 1) & ~1;
        cut = shift >= 32 ? 0u : most >> shift << shift;
        int turn = 1;
        while (shift > 0) {
            shift -= 2;
            const uint32_t t1 = cut | 1u << shift, t2 = cut | 2u << shift, t3 = cut | 3u << shift;
            uint32_t c1 = 0, c2 = 0, c3 = 0;
#pragma unroll U
            for (int i = 0; i < per_thread; i++) {
                const uint32_t k = key_at(i);
                c1 += __builtin_popcountll(__ballot(k >= t1));
                c2 += __builtin_popcountll(__ballot(k >= t2));
                c3 += __builtin_popcountll(__ballot(k >= t3));
            }
            if (lane == 0) sm[turn][wave][0] = c1, sm[turn][wave][1] = c2, sm[turn][wave][2] = c3;
            __syncthreads();
            c1 = c2 = c3 = 0;
#pragma unroll
            for (int w = 0; w < NW; w++) c1 += sm[turn][w][0], c2 += sm[turn][w][1], c3 += sm[turn][w][2];
            cut = c3 >= need ? t3 : c2 >= need ? t2 : c1 >= need ? t1 : cut;
            cut = __builtin_amdgcn_readfirstlane(cut);
            turn ^= 1;
        }
    }
    // those above the cut, the protected ones, and of the equal ones the first that there is room for
    uint32_t above = 0, equal = 0, higher = 0;
#pragma unroll U
    for (int i = 0; i < per_thread; i++) {
        const int p = first + 64 * i;
        const uint32_t k = key_at(i);
        const bool kept = p < n && (p < lo || p >= hi), more = need > 0 && k > cut;
        above += kept || more;
        higher += more;
        equal += need > 0 && k == cut;
    }
    const uint32_t both = wave_sum(above | equal << 16);
    above = both & 0xFFFFu, equal = both >> 16;
    higher = wave_sum(higher);
    __syncthreads();  // (the steps' counts are read)
    if (lane == 0) sm[0][wave][0] = above, sm[0][wave][1] = equal, sm[0][wave][2] = higher;
    __syncthreads();
    uint32_t room = need;
#pragma unroll
    for (int w = 0; w < NW; w++) room -= sm[0][w][2];
    uint32_t at = 0, ties = 0;
    for (int w = 0; w < wave; w++) {
        const uint32_t e = sm[0][w][1], take = ties < room ? min(e, room - ties) : 0u;
        at += sm[0][w][0] + take;
        ties += e;
    }
    const uint64_t below = (1ull << lane) - 1;
#pragma unroll U
    for (int i = 0; i < per_thread; i++) {
        const int p = first + 64 * i;
        const uint32_t k = key_at(i);
        const bool tie = need > 0 && k == cut;
        const uint64_t tied = __ballot(tie);
        const bool in = (p < n && (p < lo || p >= hi)) || (need > 0 && k > cut) ||
                        (tie && ties + (uint32_t)__builtin_popcountll(tied & below) < room);
        const uint64_t all = __ballot(in);
        if (in) picked[at + (uint32_t)__builtin_popcountll(all & below)] = p;
        at += (uint32_t)__builtin_popcountll(all);
        ties += (uint32_t)__builtin_popcountll(tied);
    }
}

}  // namespace

int paged_select(PagedCache& c, const PagedQuery& q, int budget, int sink, int recent, int32_t* picked, hipStream_t stream) {
    if (int rc = check_query(c, q, "paged select")) return rc;
    QW_REQUIRE(budget > 0 && sink >= 0 && recent >= 0 && (int64_t)sink + recent <= budget, QW_ERR_INVALID_ARGUMENT,
               "paged select: budget > 0 and sink + recent <= budget, neither negative, expected");
    QW_REQUIRE((int64_t)budget * c.page_size <= 0x7fffff00, QW_ERR_INVALID_ARGUMENT, "paged select: budget * page_size < 2^31 expected");
    QW_REQUIRE(q.table_width <= kMaxPages, QW_ERR_UNSUPPORTED, "paged select: at most 65536 pages a sequence");
    if (q.n_seq == 0) return QW_OK;
    QW_REQUIRE(picked, QW_ERR_INVALID_ARGUMENT, "paged select: null picked");
    QW_REQUIRE(stream != hipStreamPerThread, QW_ERR_UNSUPPORTED, "paged select: hipStreamPerThread; name a stream");
    DeviceGuard dg(c.device);
    QW_REQUIRE(dg.ok, QW_ERR_HIP, "paged select: hipSetDevice failed");
    SelectArgs a{};
    a.c = c.view;
    a.q = (const f16*)q.q;
    a.q_seq = q.seq_stride, a.q_head = q.head_stride, a.q_row = q.row_stride;
    a.lengths = q.lengths;
    a.table = q.table;
    a.table_stride = q.table_stride;
    a.width = q.table_width;
    a.G = q.n_q_heads / c.hkv;
    a.n_rows = q.n_rows;
    a.R = a.G * q.n_rows;
    a.budget = budget, a.sink = sink, a.recent = recent;
    a.picked = picked;
    if (q.table_width > budget) {
        void* ws = nullptr;
        if (int rc = workspace(kWsPagedScores, c.device, stream, (size_t)q.n_seq * c.hkv * q.table_width * 4, &ws)) return rc;
        a.scores = (float*)ws;
        // tiles of 16 pages: one a wave while that leaves CUs idle, else up to four (q's codes form once a wave). 1024 pages,
        // 8 heads, one / four, us with the pick: 1 sequence 9.5 / 11.3, 4 11.0 / 11.4, 32 29.2 / 20.9, 64 47.3 / 34.3
        const int64_t tiles = (int64_t)(q.table_width + 15) / 16 * c.hkv * q.n_seq;
        a.tiles = (int)std::max<int64_t>(1, std::min<int64_t>(4, tiles / 4096));
        const dim3 grid((unsigned)((q.table_width + 64 * a.tiles - 1) / (64 * a.tiles)), c.hkv, q.n_seq);
        if (c.D == 256)
            hipLaunchKernelGGL(paged_score_kernel<256>, grid, dim3(256), 0, stream, a);
        else
            hipLaunchKernelGGL(paged_score_kernel<128>, grid, dim3(256), 0, stream, a);
        QW_HIP_CHECK(hipGetLastError());
    }
    // scores in the registers of 256 or 1024 threads, or read again, us with the scores: 1 sequence of 1024 pages 9.5, 11.8, 10.2;
    // of 8192 (1024 threads) 16.5, 23.4; 16 of 8192 58.6, 65.3
    const dim3 grid(c.hkv, q.n_seq);
    if (q.table_width <= 2048)
        hipLaunchKernelGGL((paged_pick_kernel<256, 8>), grid, dim3(256), 0, stream, a);
    else if (q.table_width <= 8192)
        hipLaunchKernelGGL((paged_pick_kernel<1024, 8>), grid, dim3(1024), 0, stream, a);
    else
        hipLaunchKernelGGL((paged_pick_kernel<1024, 0>), grid, dim3(1024), 0, stream, a);
    QW_HIP_CHECK(hipGetLastError());
    return QW_OK;
}

}  // namespace qw
