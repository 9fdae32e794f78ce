// attend_shared.hpp - the launches of attention over a shared prefix and tails
// (attend_shared.hip), also taken by the attention that counts key weights
// (key_weights.hip: one cache, no prefix).
#pragma once

#include "kv_cache.hpp"

namespace qw {

// One cache's part of the keys.
struct SharedSegment {
    const uint32_t* k_data;
    const uint32_t* k_params;
    const uint32_t* v_data;
    const uint32_t* v_params;
    const int* fast_flag;         // device: every stored scale is in the range of the short dequantization
    int bits, cap, T;
    uint32_t code_off2;
    int heads, rows;              // the cache's heads; query rows of each
    int unit_rows;                // rows of a unit (the head's rows in equal query tiles)
    int n_split, tiles_per_split;
    int n_units;                  // heads * query tiles * n_split; 0: no such keys
    int slot0;                    // its first split's partial slot
    int causal_rows;              // > 0: of that many last rows, row r sees keys to T - causal_rows + r
};

struct SharedArgs {
    const f16* q;           // [n_seq][hkv * G][Tq][D]
    f16* out;               // like q; written directly where n_slots == 1
    float* part_o;          // [n_slots][hkv][R][D], dims in order
    float2* part_ml;        // [n_slots][hkv][R]: the maximum in log2 units, the sum
    const int32_t* starts;  // [n_seq] or null: a sequence's first tail key
    int Tq, G, hkv, R;      // R = n_seq * Tq * G: row (b * Tq + r) * G + head in group
    int n_slots;
    float* scores;          // null, or [hkv][R][score_stride]: the scores (log2 units) of one cache's few rows
    int64_t score_stride;   // a multiple of 32
    float scale2;           // |scale| * log2 e
    uint32_t q_flip;        // the sign bits of two halves where scale is negative: q is taken negated
    SharedSegment seg[2];   // the prefix, the tails
};

// Dims of a K row that a lane group g (lane >> 4) holds as a QK operand: 16-byte pieces 4 i + g of
// the row's codes, so that one load of a wave takes 64 whole bytes of each of 16 rows (pieces of one
// group side by side took each line four to eight times over from a cache that holds none of them
// that long). Step m then multiplies dims 8 k_chunk(m, g) .. + 7, E = 16 / KIND steps a piece, and
// piece i's scale is of group k_piece_group(i, g).
template <int KIND>
__host__ __device__ constexpr int k_chunk(int m, int g) {
    constexpr int E = 16 / KIND;
    return E * (4 * (m / E) + g) + m % E;
}
template <int KIND>
__host__ __device__ constexpr int k_piece_group(int i, int g) {
    return KIND == 16 ? 0 : KIND == 8 ? i : 2 * i + g / 2;
}

constexpr int kSharedMaxSlots = 512;
__host__ __device__ constexpr int shared_tile(int D) { return 16384 / D; }  // keys of a split's tile
constexpr int kSharedLds = 146 * 1024;  // a workgroup's

// Fills the arguments and takes the workspace (either cache may be null); the launches.
int plan_shared(const KVCache* prefix, const KVCache* tails, const void* q, int n_seq, int n_rows, int G, int hkv,
                const int32_t* starts, float scale, bool causal, void* out, hipStream_t stream, SharedArgs* a);
int launch_shared(const KVCache* prefix, const KVCache* tails, const SharedArgs& a, hipStream_t stream);
int launch_shared_merge(int D, const SharedArgs& a, hipStream_t stream);

// A row's partials joined by a workgroup of 256: D / 4 threads a partial row, 1024 / D partial rows
// at a time and four such in flight, their sums over LDS.
template <int D>
struct SharedMerge {
    float4v o[256];
    float l[1024 / D];
};
template <int D>
__device__ __forceinline__ void merge_row(const SharedArgs& a, int row, int h, SharedMerge<D>& sm) {
    constexpr int LPR = D / 4, NS = 256 / LPR, AHEAD = 4;
    const int tid = threadIdx.x, c = tid % LPR, s0 = tid / LPR;
    const int64_t stride = (int64_t)a.hkv * a.R, at = (int64_t)h * a.R + row;
    float M = -INFINITY;
    for (int s = tid & 63; s < a.n_slots; s += 64) M = fmaxf(M, a.part_ml[s * stride + at].x);
    M = wave_reduce(M, OpMax{});
    const float mr = M == -INFINITY ? 0.0f : M;
    float4v o = {0.f, 0.f, 0.f, 0.f};
    float l = 0.0f;
    for (int s = s0; s < a.n_slots; s += NS * AHEAD) {
        float2 ml[AHEAD];
        float4v x[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const int64_t p = min(s + NS * i, a.n_slots - 1) * stride + at;
            ml[i] = a.part_ml[p];
            x[i] = *(const float4v*)(a.part_o + p * D + 4 * c);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            if (s + NS * i >= a.n_slots) break;
            const float f = __builtin_amdgcn_exp2f(ml[i].x - mr);
            l += f * ml[i].y;
#pragma unroll
            for (int j = 0; j < 4; j++) o[j] += f * x[i][j];
        }
    }
    sm.o[tid] = o;
    if (c == 0) sm.l[s0] = l;
    __syncthreads();
    if (s0 > 0) return;
#pragma unroll
    for (int s = 1; s < NS; s++) {
        const float4v x = sm.o[s * LPR + c];
#pragma unroll
        for (int j = 0; j < 4; j++) o[j] += x[j];
        l += sm.l[s];
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int seq = row / (a.Tq * a.G), rr = row % (a.Tq * a.G);
    half4v y;
#pragma unroll
    for (int j = 0; j < 4; j++) y[j] = (f16)(o[j] * inv);
    *(half4v*)(a.out + (((int64_t)seq * a.hkv * a.G + h * a.G + rr % a.G) * a.Tq + rr / a.G) * D + 4 * c) = y;
}

}  // namespace qw
