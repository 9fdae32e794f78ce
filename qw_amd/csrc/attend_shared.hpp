// attend_shared.hpp - the launches of attention over a shared prefix and tails
// (attend_shared.hip), also taken by the attention that counts key weights
// (key_weights.hip: one cache, no prefix).
#pragma once

#include "kv_cache.hpp"

namespace qw {

// A Turbo4 cache: q rotated into the K basis by a launch before, keys and values as the expansion holds
// them (f16(centroid * rescale)), the output rotated back out of the V basis by a launch behind.

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
    const float* t4_cb;           // Turbo4 caches: the 16 centroids on the device, else null
    const char* images;           // null, or its key tiles dequantized (the tails alone): [heads][n_tiles]
    int n_tiles;
    int causal_rows;              // > 0: of that many last rows, row r sees keys to T - causal_rows + r
};

struct SharedArgs {
    const f16* q;           // [n_seq][hkv * G][Tq][D]
    f16* out;               // like q; written directly where n_slots == 1
    float* part_o;          // [n_slots][hkv][R][D], a row's pieces of 4 dims as part_dim has them
    float2* part_ml;        // [n_slots][hkv][R]: the maximum in log2 units, the sum
    const int32_t* starts;  // [n_seq] or null: a sequence's first tail key
    int Tq, G, hkv, R;      // R = n_seq * Tq * G: row (b * Tq + r) * G + head in group
    int n_slots;
    float2* row_ml;         // null, or [hkv][R]: the merge leaves a row's maximum (log2 units) and 1 / its sum
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

// The first of the 4 dims at piece `place` of a partial row. The lanes that hold a row have D / 16 dims each; a
// store of the first four of all 16 lanes, then of the next, writes runs of 256 bytes. (Dims in order,
// 16 bytes every 64: 16 sequences over 32k 4-bit keys 37.0 for 31.4 us, 18.6 MB of partials.)
template <int D>
__device__ __forceinline__ int part_dim(int place) {
    return 4 * (place % 16 * (D / 64) + place / 16);
}

constexpr int kSharedMaxSlots = 512;
__host__ __device__ constexpr int shared_tile(int D) { return 16384 / D; }  // keys of a split's tile
constexpr int kSharedLds = 146 * 1024;  // a workgroup's

// Makes room for n_rows more rows, so that the append that follows moves no buffer; refused while
// the stream is captured where that needs memory.
int make_room(KVCache& c, int n_rows, hipStream_t stream);
// Fills the arguments, the tails (or the one cache) taken as tail_rows long, and takes the workspace
// (either cache may be null); the launches.
int plan_shared(const KVCache* prefix, const KVCache* tails, int tail_rows, const void* q, int n_seq, int n_rows, int G,
                int hkv, const int32_t* starts, float scale, bool causal, void* out, hipStream_t stream, SharedArgs* a);
int launch_shared(const KVCache* prefix, const KVCache* tails, const SharedArgs& a, hipStream_t stream);
int launch_shared_merge(int D, const SharedArgs& a, hipStream_t stream);
// Over Turbo4 caches (c: one of them): a.q becomes the rotated q and a.out the rotated output's place, in
// the stream's workspace; rotate_out writes the rows to out.
int shared_turbo4_room(const KVCache& c, int64_t q_rows, hipStream_t stream, SharedArgs* a);
int shared_turbo4_rotate_q(const KVCache& c, const void* q, int64_t q_rows, const SharedArgs& a, hipStream_t stream);

// Rows' partials joined by workgroups of 256, each partial row by TC threads and SG of them at a
// time, four such in flight, their sums over LDS. A workgroup a row (TC = D / 4), but: few rows of
// many slots are cut into 64 dims a workgroup, and of many rows of few slots a workgroup takes 1024 / D.
// D = 256, a row / cut: 24 rows of 45 slots 4.2 / 3.3 us, of 16 3.2 / 3.1, 512 of 45 6.9 / 7.4, of 128 21.7 / 18.8, 1024
// of 128 26 / 34; a row / several: 4096 rows of 3 slots 5.9 / 4.6, of 8 9.6 / 8.6, 2048 of 3 3.9 / 3.7, of 8 5.5 / 5.7, 32768 of
// 8 56 / 58, of 12 76 / 87.
enum MergeForm { kMergeRow, kMergeCut, kMergeRows };
__host__ __device__ inline MergeForm merge_form(int64_t rows, int n_slots) {
    return n_slots > 16 && rows <= 512 ? kMergeCut : n_slots <= 8 && rows >= 4096 ? kMergeRows : kMergeRow;
}
__host__ __device__ inline int merge_groups(int D, int R, int hkv, int n_slots) {
    const MergeForm f = merge_form((int64_t)R * hkv, n_slots);
    return f == kMergeCut ? R * (D / 64) : f == kMergeRow ? R : (R + 1024 / D - 1) / (1024 / D);
}
struct SharedMerge {
    float4v o[256];
    float l[16];
};
template <int D, int SG, int TC>
__device__ __forceinline__ void merge_rows(const SharedArgs& a, int group, int h, SharedMerge& sm) {
    constexpr int AHEAD = 4, CUTS = SG == 1 ? 1 : D / 4 / TC;  // workgroups a row
    const int tid = threadIdx.x, sg = SG == 1 ? 0 : tid / TC;
    const int row = SG == 1 ? group * (256 / TC) + tid / TC : group / CUTS;
    const int c = group % CUTS * TC + tid % TC;
    if (row >= a.R) return;  // (SG == 1: no barrier follows)
    const int64_t stride = (int64_t)a.hkv * a.R, at = (int64_t)h * a.R + row;
    float M = -INFINITY;
    if constexpr (SG == 1) {
        for (int s = 0; s < a.n_slots; s++) M = fmaxf(M, a.part_ml[s * stride + at].x);
    } else {
        for (int s = tid & 63; s < a.n_slots; s += 64) M = fmaxf(M, a.part_ml[s * stride + at].x);
        M = wave_reduce(M, OpMax{});
    }
    const float mr = M == -INFINITY ? 0.0f : M;
    float4v o = {0.f, 0.f, 0.f, 0.f};
    float l = 0.0f;
    for (int s = sg; s < a.n_slots; s += SG * AHEAD) {
        float2 ml[AHEAD];
        float4v x[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const int64_t p = min(s + SG * i, a.n_slots - 1) * stride + at;
            ml[i] = a.part_ml[p];
            x[i] = *(const float4v*)(a.part_o + p * D + 4 * c);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            if (s + SG * i >= a.n_slots) break;
            const float f = __builtin_amdgcn_exp2f(ml[i].x - mr);
            l += f * ml[i].y;
#pragma unroll
            for (int j = 0; j < 4; j++) o[j] += f * x[i][j];
        }
    }
    if constexpr (SG > 1) {
        sm.o[tid] = o;
        if (tid % TC == 0) sm.l[sg] = l;
        __syncthreads();
        if (sg > 0) return;
#pragma unroll
        for (int s = 1; s < SG; s++) {
            const float4v x = sm.o[s * TC + tid];
#pragma unroll
            for (int j = 0; j < 4; j++) o[j] += x[j];
            l += sm.l[s];
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (a.row_ml && c == 0) a.row_ml[at] = float2{mr, inv};
    const int seq = row / (a.Tq * a.G), rr = row % (a.Tq * a.G);
    half4v y;
#pragma unroll
    for (int j = 0; j < 4; j++) y[j] = (f16)(o[j] * inv);
    *(half4v*)(a.out + (((int64_t)seq * a.hkv * a.G + h * a.G + rr % a.G) * a.Tq + rr / a.G) * D + part_dim<D>(c)) = y;
}
template <int D>
__device__ __forceinline__ void merge_group(const SharedArgs& a, int group, int h, SharedMerge& sm) {
    const MergeForm f = merge_form((int64_t)a.R * a.hkv, a.n_slots);
    if (f == kMergeCut)
        merge_rows<D, 16, 16>(a, group, h, sm);
    else if (f == kMergeRow)
        merge_rows<D, 1024 / D, D / 4>(a, group, h, sm);
    else
        merge_rows<D, 1, D / 4>(a, group, h, sm);
}

}  // namespace qw
