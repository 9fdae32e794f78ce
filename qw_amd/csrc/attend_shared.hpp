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
    int cap, T;
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
    float scale2;           // scale * log2 e
    SharedSegment seg[2];   // the prefix, the tails
};

constexpr int kSharedMaxSlots = 512;

// Fills the arguments and takes the workspace (either cache may be null); the launches.
int plan_shared(const KVCache* prefix, const KVCache* tails, const void* q, int n_seq, int n_rows, int G, int hkv,
                const int32_t* starts, float scale, bool causal, void* out, hipStream_t stream, SharedArgs* a);
int launch_shared(const KVCache* prefix, const KVCache* tails, const SharedArgs& a, hipStream_t stream);
int launch_shared_merge(int D, const SharedArgs& a, hipStream_t stream);

}  // namespace qw
