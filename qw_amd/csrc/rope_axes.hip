// rope_axes.hip - rotary positions of several axes (time, height, width) for packed tokens.
//
// Pair p of a head's first rope_dims dims turns by positions[axes[p]][token] * scale * base^(-p / half):
//   r1 = x1 cos - x2 sin,  r2 = x1 sin + x2 cos
// with the angle reduced in 64 bits (turns modulo one), so that far positions keep theirs: in fp32 a
// position of 10^6 is off by up to 0.06 radians. A workgroup forms its tokens' cosines and sines once, in
// LDS, for all heads; then it is a copy, bound by reading and writing q and k (32768 tokens of 32 + 8 heads, D = 128:
// 134 us, 5.0 TB/s; a large copy 5.1).
#include <algorithm>
#include <cmath>

#include "paged.hpp"
#include "rope.hpp"

namespace qw {

namespace {

constexpr int kAngles = 2048;   // (cos, sin) of a workgroup

struct RopeAxesArgs {
    const f16* qkv;
    f16* q_out;
    f16* k_out;
    RopeTurns r;
    int n, hq, hkv, D, tokens;  // tokens of a workgroup
};

// VEC: 8 dims a thread (head_dim and half multiples of 8), else one.
template <bool VEC>
__global__ __launch_bounds__(256) void rope_axes_kernel(RopeAxesArgs a) {
    __shared__ float2 sm[kAngles];
    const int t0 = blockIdx.x * a.tokens, nt = min(a.tokens, a.n - t0);
    const int half = a.r.half, traditional = a.r.traditional;
    for (int p = threadIdx.x % 64; p < half; p += 64) {
        const double f = turn_rate(a.r, p);
        const int32_t* pos = a.r.positions + a.r.axes[p] * a.r.stride + t0;
        for (int t = threadIdx.x / 64; t < nt; t += 4) sm[t * half + p] = turn_of(f, pos[t]);
    }
    __syncthreads();
    constexpr int N = VEC ? 8 : 1;
    const int per = a.D / N, heads = a.hq + a.hkv, R = 2 * half;
    const int total = nt * heads * per;
    for (int i = threadIdx.x; i < total; i += 256) {
        const int d = i % per * N, row = i / per, t = row / heads, h = row - t * heads;
        const int64_t token = t0 + t;
        const f16* in = a.qkv + (token * (heads + a.hkv) + h) * a.D;
        f16* out = h < a.hq ? a.q_out + (token * a.hq + h) * a.D : a.k_out + (token * a.hkv + h - a.hq) * a.D;
        alignas(16) f16 x[N], y[N];
        if constexpr (VEC)
            *(half8*)x = *(const half8*)(in + d);
        else
            x[0] = in[d];
        if (d >= R) {
#pragma unroll
            for (int e = 0; e < N; e++) y[e] = x[e];
        } else {
            const bool first = traditional ? true : d < half;
            alignas(16) f16 z[N];  // the other dims of its pairs
            if (traditional) {
#pragma unroll
                for (int e = 0; e < N; e++) z[e] = VEC ? x[e ^ (N > 1)] : in[d ^ 1];
            } else if constexpr (VEC) {
                *(half8*)z = *(const half8*)(in + (first ? d + half : d - half));
            } else {
                z[0] = in[first ? d + half : d - half];
            }
#pragma unroll
            for (int e = 0; e < N; e++) {
                const bool one = traditional ? ((d + e) & 1) == 0 : first;
                const int p = traditional ? (d + e) >> 1 : first ? d + e : d + e - half;
                const float2 cs = sm[t * half + p];
                float r1, r2;
                rope_rot((float)(one ? x[e] : z[e]), (float)(one ? z[e] : x[e]), cs.x, cs.y, r1, r2);
                y[e] = (f16)(one ? r1 : r2);
            }
        }
        if constexpr (VEC)
            // (past the caches: 4099 tokens of 24 + 4 heads, D = 256, 24.5 us, so 20.9)
            __builtin_nontemporal_store(*(const half8*)y, (half8*)(out + d));
        else
            out[d] = y[0];
    }
}

}  // namespace

int rope_turns(const RopeAxes& r, int n_tokens, int hq, int hkv, int D, RopeTurns& out) {
    QW_REQUIRE(n_tokens >= 0 && n_tokens <= (1 << 28) && hq > 0 && hkv > 0 && D > 0 && (int64_t)hq + 2 * (int64_t)hkv <= (1 << 24) / D,
               QW_ERR_INVALID_ARGUMENT, "rope axes: 0 .. 2^28 tokens, n_q_heads, n_kv_heads and head_dim > 0, a row of at most 2^24 values expected");
    QW_REQUIRE(r.rope_dims > 0 && r.rope_dims % 2 == 0 && r.rope_dims <= D && r.rope_dims <= 2 * kMaxHalf && D % 2 == 0,
               QW_ERR_INVALID_ARGUMENT, "rope axes: rope_dims even, positive, at most head_dim and 512, head_dim even");
    QW_REQUIRE(r.base > 0.0f && std::isfinite(r.base) && std::isfinite(r.scale), QW_ERR_INVALID_ARGUMENT,
               "rope axes: a finite base > 0 and a finite scale expected");
    QW_REQUIRE(r.n_axes > 0 && r.axes && r.stride >= n_tokens, QW_ERR_INVALID_ARGUMENT,
               "rope axes: n_axes > 0, an axis for each pair, and a positions stride of n_tokens at least expected");
    for (int p = 0; p < r.rope_dims / 2; p++) {
        QW_REQUIRE(r.axes[p] < r.n_axes, QW_ERR_INVALID_ARGUMENT, "rope axes: a pair's axis is not below n_axes");
        out.axes[p] = r.axes[p];
    }
    out.positions = r.positions;
    out.stride = r.stride;
    out.half = r.rope_dims / 2;
    out.traditional = r.traditional;
    out.log2_base = std::log2((double)r.base);
    out.scale = (double)r.scale / 6.283185307179586476925;
    return QW_OK;
}

int rope_axes(const RopeAxes& r, const void* qkv, int n_tokens, int hq, int hkv, int D, void* q_out, void* k_out,
              hipStream_t stream) {
    RopeAxesArgs a{};
    if (int rc = rope_turns(r, n_tokens, hq, hkv, D, a.r)) return rc;
    if (n_tokens == 0) return QW_OK;
    QW_REQUIRE(qkv && q_out && k_out && r.positions, QW_ERR_INVALID_ARGUMENT, "rope axes: null qkv/positions/output");
    a.qkv = (const f16*)qkv;
    a.q_out = (f16*)q_out;
    a.k_out = (f16*)k_out;
    a.n = n_tokens, a.hq = hq, a.hkv = hkv, a.D = D;
    // a token a workgroup while there are few, else as many as its angles' place holds, up to 8. One / 8, 32 + 8 heads of
    // D = 128, replayed, us: 64 tokens 5.2 / 18.8, 1500 9.1 / 19.5, 4099 18.2 / 25.7, 32768 141 / 134
    a.tokens = std::max(1, std::min({8, n_tokens / 4096, kAngles / a.r.half}));
    const int64_t groups = ((int64_t)n_tokens + a.tokens - 1) / a.tokens;
    QW_REQUIRE(groups * 256 <= UINT32_MAX, QW_ERR_UNSUPPORTED, "rope axes: too many tokens for one call");
    const dim3 grid((unsigned)groups);
    const bool vec = D % 8 == 0 && a.r.half % 8 == 0 && ((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)k_out) % 16 == 0;
    if (vec)
        hipLaunchKernelGGL(rope_axes_kernel<true>, grid, dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL(rope_axes_kernel<false>, grid, dim3(256), 0, stream, a);
    QW_HIP_CHECK(hipGetLastError());
    return QW_OK;
}

int paged_rope_update(PagedCache& c, const RopeAxes& r, const void* qkv, int hq, void* q_out, const PagedSeqs& s,
                      hipStream_t stream) {
    if (int rc = check_seqs(c, s, "paged rope update")) return rc;
    QW_REQUIRE((uintptr_t)qkv % 8 == 0, QW_ERR_INVALID_ARGUMENT, "paged rope update: qkv 8-byte aligned expected");
    DeviceGuard dg(c.device);
    QW_REQUIRE(dg.ok, QW_ERR_HIP, "paged rope update: hipSetDevice failed");
    if (s.n_tokens == 0) return rope_axes(r, qkv, 0, hq, c.hkv, c.D, q_out, nullptr, stream);
    // One launch for a step of few sequences: each workgroup forms its tokens' angles anew, one token behind the other. Two launches /
    // one, replayed, us: 24 heads over 4, D = 256, 1 token 9.8 / 6.6, 64 of 64 sequences 10.3 / 7.2, 256 of 256 11.6 / 8.2, 256 of 8
    // 12.7 / 13.7, 1024 of 1024 19.8 / 21.0; 32 over 8, D = 128, 256 of 256 11.3 / 9.7, 256 of 8 14.4 / 20.3.
    if (s.n_tokens <= std::min(256, s.n_seq) && r.rope_dims % 8 == 0 && (uintptr_t)q_out % 8 == 0) {
        RopeTurns t;
        if (int rc = rope_turns(r, s.n_tokens, hq, c.hkv, c.D, t)) return rc;
        return paged_turn_update(c, t, qkv, hq, q_out, s, stream);
    }
    // the rotated keys pass through a workspace on their way into the pages (one handle, a stream a thread: they would share it)
    QW_REQUIRE(stream != hipStreamPerThread, QW_ERR_UNSUPPORTED, "paged rope update: hipStreamPerThread; name a stream");
    void* k = nullptr;
    if (int rc = workspace(kWsPagedKeys, c.device, stream, (size_t)s.n_tokens * c.hkv * c.D * sizeof(f16), &k)) return rc;
    if (int rc = rope_axes(r, qkv, s.n_tokens, hq, c.hkv, c.D, q_out, k, stream)) return rc;
    const int64_t row = (int64_t)(hq + 2 * c.hkv) * c.D;
    return paged_update(c, k, (const f16*)qkv + (int64_t)(hq + c.hkv) * c.D, (int64_t)c.hkv * c.D, c.D, row, c.D, s, stream);
}

}  // namespace qw
