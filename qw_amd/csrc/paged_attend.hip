// paged_attend.hip - attention of the newest tokens of many sequences over their pages.
//
// out = softmax(scale q . k) v for each row over its sequence's keys, causal among the last n_rows of
// them, in one pass with the running maximum and sum. Bound by reading the codes once from HBM: 64 sequences of
// up to 16k fp16 keys (8 KV heads, D = 128) 435 us, 6.6 TB/s; one of 128k keys 5.0 to 5.8 TB/s in every mode. Short ones are bound by their start (lengths, table, queries and keys, one behind the other, 4 us), the
// last joining and the second launch (4 us).
//
// Work is dealt in rounds of 128 or 256 keys to the workers of a head (a grid sized for the card, lengths read on the
// device): short sequences one by one, else pieces of one sequence each or, if that does not come out even, the
// rounds of all sequences, one behind the other, in equal runs. So sequences of any lengths keep the chip busy. A
// worker's piece of a sequence that is not all of it goes to a workspace as fp32 partials that a second launch joins.
//
// A wave takes 32 keys of a round, by DMA through an LDS place of its own (fp16 keys through registers) and, as they
// lie, into the matrix instructions' operands:
//   S^T = K Q^T: two tiles of 16 keys; tile t's row i is key 8 (i / 4) + 4 t + i % 4, so that lane
//     group g ends with the scores of keys 8 g .. 8 g + 7 of the query row that it holds, which is
//   O^T = V^T P^T's second operand as it stands; V's 8 codes of a dim are the first.
// Codes enter as subnormal halves (paged.hpp). A group's score is scale * (q . code) + bias * sum q; P
// is multiplied by a key's V scale in fp32 and rounded once to fp16, P'. With the codes' middle c0,
//   sum_k P (scale code + bias) = sum_k P' code - c0 sum_k P' + sum_k P (bias + c0 scale):
// one more matrix product each for the last two. So P's and P's rounding meet what is left of a code beside the middle, not
// the code and the bias that nearly cancel each other (17 sequences of 4 bits: an error of 0.00028 of the result for 0.00069,
// for 0.9 us of 32). P is rounded because the matrix instructions take halves; a product of more bits costs two of them. Of
// the 0.00028 the result's own rounding is 0.00021.
// The next round's K is requested behind this one's scores, its V behind this one's P V, into the place that they
// leave: a wave always waits for loads that are half a round old, and never for another wave.
#include <algorithm>

#include "paged.hpp"

namespace qw {

namespace {

constexpr float kNone = -0x1p100f;      // a maximum below every score
constexpr float kLazy = 4.0f;           // scores pass the reference by so much (log2) before it follows
constexpr float kLift = 10.0f;          // log2 of P at the reference: P <= 2^14, times a scale below 2, fits a half

struct AttendArgs {
    PagedView c;
    const f16* q;
    int64_t q_seq, q_head, q_row;
    f16* out;
    const int32_t* lengths;
    const int32_t* table;
    int64_t table_stride;
    int width, n_seq, G, n_rows, R;  // R = G * n_rows rows of a KV head: row g * n_rows + r
    const int32_t* picked;
    int n_picked;
    float scale2;  // scale * log2 e
    int workers, round;  // keys of a round: 32 a wave
    int whole;           // sequence by sequence, worker b % workers' each, and no second launch follows
    float* part_o;    // [2 workers][hkv][R][D]
    float2* part_ml;  // [2 workers][hkv][R]
    uint4* cut;       // above 64 sequences, for each worker: the one whose first piece ends its run, unfinished (or -1),
                      // the rounds before it, its own, and all
};

// A sequence's keys as the kernel walks them: the whole of it, or its picked pages side by side.
__device__ __forceinline__ int keys_of(const AttendArgs& a, int len) {
    if (!a.picked) return len;
    const int pages = (len + (1 << a.c.lg) - 1) >> a.c.lg;
    return min(pages, a.n_picked) << a.c.lg;
}
__device__ __forceinline__ uint32_t rounds_of(const AttendArgs& a, int b) {
    return (uint32_t)(keys_of(a, min(max(a.lengths[b], 0), a.width << a.c.lg)) + a.round - 1) / a.round;
}

// How the rounds are dealt, the same for every wave of a call. Up to 64 sequences (a lane each): pieces of
// one sequence each, of at most `most` rounds, one a worker, if there is such a length not much above the
// average; a second piece would begin with its own loads, one behind the other. Else equal runs of all rounds.
struct Plan {
    int len;                            // lane b's sequence (up to 64)
    uint32_t rounds, through;           // its rounds, and all up to it
    uint32_t total, workers, per, rest; // the first `rest` runs have per + 1 rounds
    uint32_t most, pieces, last;        // piece by piece: its pieces, and all up to it; else most = 0
};
__device__ __forceinline__ uint32_t wave_last(uint32_t x) { return (uint32_t)__builtin_amdgcn_readlane((int)x, 63); }
__device__ __forceinline__ Plan plan_of(const AttendArgs& a) {
    const int lane = (int)__lane_id();
    Plan p{};
    if (a.n_seq <= 64) {
        if (lane < a.n_seq) {
            p.len = min(max(a.lengths[lane], 0), a.width << a.c.lg);
            p.rounds = (uint32_t)(keys_of(a, p.len) + a.round - 1) / a.round;
        }
        p.through = wave_scan(p.rounds);
        p.total = wave_last(p.through);
    } else {
        uint32_t n = 0;
#pragma unroll 8
        for (int b0 = 0; b0 < a.n_seq; b0 += 64) {
            const uint32_t c = rounds_of(a, min(b0 + lane, a.n_seq - 1));
            n += b0 + lane < a.n_seq ? c : 0u;
        }
        p.total = wave_last(wave_scan(n));
    }
    p.workers = min((uint32_t)a.workers, p.total);  // (a round at least for each that works)
    if (p.total == 0) return p;
    p.per = __builtin_amdgcn_readfirstlane(p.total / p.workers);
    p.rest = p.total - p.per * p.workers;
    if (a.n_seq <= 64) {
        uint32_t most = p.per + (p.rest > 0);
        for (int i = 0; i < 4; i++, most += 1 + most / 16) {
            p.pieces = (p.rounds + most - 1) / most;
            p.last = wave_scan(p.pieces);
            if (wave_last(p.last) <= (uint32_t)a.workers) {
                p.most = most;
                break;
            }
        }
    }
    return p;
}
// Rounds r0 .. r1 - 1 of sequence b's `all`, whose partials have their place; b = -1: none.
struct Piece {
    int b, len;
    uint32_t r0, r1, all, slot;
};
// Worker w's piece that begins at round `at` of its run.
__device__ __forceinline__ Piece piece_of(const AttendArgs& a, uint32_t per, uint32_t rest, uint32_t w, uint32_t at, int b, int len,
                                          uint32_t all, uint32_t before) {
    const uint32_t begin = w * per + min(w, rest), end = begin + per + (w < rest);
    return Piece{b, len, at - before, min(all, end - before), all, 2 * w + (at == before && at != begin ? 1 : 0)};
}
// (among the sequences from b0 on, before which lie `base` rounds)
__device__ __forceinline__ Piece piece_from(const AttendArgs& a, uint32_t per, uint32_t rest, uint32_t w, uint32_t at, int b0, uint32_t base) {
    const PagedUnit u = find_unit(a.n_seq, at, [&](int b) { return rounds_of(a, b); }, b0, base);
    if (u.b < 0) return Piece{-1, 0, 0, 0, 0, 0};
    return piece_of(a, per, rest, w, at, u.b, min(max(a.lengths[u.b], 0), a.width << a.c.lg), rounds_of(a, u.b), u.base);
}
// Its first piece (piece by piece: its only one); at: the round that it begins with.
__device__ __forceinline__ Piece first_piece(const AttendArgs& a, const Plan& p, uint32_t w, uint32_t at) {
    if (a.n_seq > 64) return piece_from(a, p.per, p.rest, w, at, 0, 0u);
    const uint64_t past = __ballot(p.most ? p.last > w : p.through > at);
    if (!past) return Piece{-1, 0, 0, 0, 0, 0};
    const int b = __builtin_ctzll(past);
    const int len = __builtin_amdgcn_readlane(p.len, b);
    const uint32_t all = (uint32_t)__builtin_amdgcn_readlane((int)p.rounds, b);
    if (p.most) {
        const uint32_t n = (uint32_t)__builtin_amdgcn_readlane((int)p.pieces, b);
        const uint32_t i = w - ((uint32_t)__builtin_amdgcn_readlane((int)p.last, b) - n);
        const uint32_t each = __builtin_amdgcn_readfirstlane(all / n), more = all - each * n;
        const uint32_t r0 = i * each + min(i, more);
        return Piece{b, len, r0, r0 + each + (i < more), all, 2 * w};
    }
    return piece_of(a, p.per, p.rest, w, at, b, len, all, (uint32_t)__builtin_amdgcn_readlane((int)p.through, b) - all);
}

// 32 keys' place: of each 16 the pool's page, the slot, and the position of the first.
struct Place {
    int page0, page1, slot0, slot1, pos0, pos1;
};
// The places of a wave's keys in 32 rounds, a lane each 16 keys: a round's come by two lane reads. (As scalar loads round
// by round they shared a counter with the queries' LDS reads, which then waited for them.)
struct Places {
    int page, pos;
};
constexpr int kNoKey = 0x7fffff00;  // a position behind every key

// How a call's row tiles of 16 go to waves: up to 16 rows a tile and 4 waves a workgroup; above, two tiles, for both of
// which a wave takes its keys once, and 8 waves that share the queries. fp16 keys go through registers, but for two tiles
// at D = 256: there 4 waves fill LDS.
template <int BITS, int D, int TILES>
struct Form {
    static constexpr bool WIDE = BITS == 16 && D == 256 && TILES == 2;
    static constexpr bool RING = BITS != 16 || WIDE;         // keys come through LDS
    static constexpr int WAVES = WIDE ? 4 : 4 * TILES;
    static constexpr int SIMD = WIDE ? 1 : D == 128 && TILES == 1 ? (RING ? 4 : 3) : 2;  // waves a SIMD that the registers are cut for
    static constexpr int ROUND = 32 * WAVES;
};

template <int BITS, int D, bool INT8>
struct Shape {
    static constexpr int NG = INT8 ? 1 : D / kGroup;
    static constexpr int NK = D * BITS / 512;               // 16-byte pieces of a K row a lane group
    static constexpr int DPP = BITS == 16 ? 1 : 16 / BITS;  // dims of a V piece
    static constexpr int NV = D / 16 / DPP;
    static constexpr int PAR = BITS == 16 ? 0 : INT8 ? 8 : 16 * NG;  // halves of 8 keys' scales and biases
    // A wave's 32 keys in LDS, each of its loads' 1 KB as the lanes hold it: K, V, K's and V's scales and biases.
    static constexpr int V0 = 2 * NK * 1024, P0 = V0 + NV * 1024, SLOT = P0 + (PAR ? 1024 : 0);
    static constexpr int K_LOADS = 2 * NK + (PAR ? 1 : 0), V_LOADS = NV + (PAR ? 1 : 0);
};

// One load of 64 times 16 bytes to LDS. M0, which gives the place, is saved and restored so that the compiler's
// view of it holds; the offset counts for both addresses. The compiler knows nothing of the load: what reads the
// place waits by wait_loads first.
#define QW_TO_LDS(CACHE)                                            \
    asm volatile(                                                   \
        "s_mov_b32 %0, m0\n\t"                                      \
        "s_mov_b32 m0, %2\n\t"                                      \
        "s_nop 0\n\t"                                               \
        "global_load_lds_dwordx4 %1, off offset:%3" CACHE "\n\t"    \
        "s_nop 0\n\t"                                               \
        "s_mov_b32 m0, %0"                                          \
        : "=&s"(saved)                                              \
        : "v"(from), "s"(__builtin_amdgcn_readfirstlane(place - OFFSET)), "n"(OFFSET) \
        : "memory")
template <int OFFSET, bool PAST>
__device__ __forceinline__ void to_lds(const char* from, uint32_t place) {
    uint32_t saved;
    if constexpr (PAST)
        QW_TO_LDS(" nt");
    else
        QW_TO_LDS("");
}
#undef QW_TO_LDS
template <int N, int STEP, bool PAST, int J = 0>
__device__ __forceinline__ void run_to_lds(const char* from, uint32_t place) {
    if constexpr (J < N) {
        to_lds<J * STEP, PAST>(from, place + J * 1024);
        run_to_lds<N, STEP, PAST, J + 1>(from, place);
    }
}
template <int N>
__device__ __forceinline__ void wait_loads() {  // until at most N of the wave's loads are on their way
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

__device__ __forceinline__ const char* k_row(const PagedView& c, const Place& p, int h, int lane, int row_bytes) {
    const int64_t page = lane & 8 ? p.page1 : p.page0;
    const int slot = (lane & 8 ? p.slot1 : p.slot0) + 8 * (lane >> 2 & 1) + (lane & 3);
    return c.k + (((page * c.hkv + h) << c.lg) + slot) * row_bytes + 16 * (lane >> 4);
}
// The 8 keys of a lane group: their place among the pool's blocks of 8.
__device__ __forceinline__ int64_t block_of(const PagedView& c, const Place& p, int h, int g) {
    const int64_t page = g & 2 ? p.page1 : p.page0;
    return ((page * c.hkv + h) << (c.lg - 3)) + ((g & 2 ? p.slot1 : p.slot0) >> 3) + (g & 1);
}

template <int BITS, int D, bool INT8, bool PAST>
__device__ __forceinline__ void params_to_lds(const PagedView& c, const f16* par, const Place& p, int h, int lane, uint32_t place) {
    constexpr int LPB = Shape<BITS, D, INT8>::PAR / 8;  // lanes of 8 keys' scales and biases
    if constexpr (LPB > 0) {
        if (lane < 4 * LPB)
            to_lds<0, PAST>((const char*)(par + block_of(c, p, h, lane / LPB) * (8 * LPB)) + lane % LPB * 16, place);
    }
}
template <int BITS, int D, bool INT8, bool PAST>
__device__ __forceinline__ void request_k(const PagedView& c, const Place& p, int h, int lane, uint32_t slot) {
    using S = Shape<BITS, D, INT8>;
    constexpr int ROW = D * BITS / 8;
    const char* row = k_row(c, p, h, lane, ROW);
    run_to_lds<S::NK, 64, PAST>(row, slot);
    run_to_lds<S::NK, 64, PAST>(row + 4 * ROW, slot + S::NK * 1024);
    params_to_lds<BITS, D, INT8, PAST>(c, c.k_par, p, h, lane, slot + S::P0);
}
template <int BITS, int D, bool INT8, bool PAST>
__device__ __forceinline__ void request_v(const PagedView& c, const Place& p, int h, int lane, uint32_t slot) {
    using S = Shape<BITS, D, INT8>;
    run_to_lds<S::NV, 256, PAST>(c.v + block_of(c, p, h, lane >> 4) * (D * BITS) + 16 * (lane & 15), slot + S::V0);
    params_to_lds<BITS, D, INT8, PAST>(c, c.v_par, p, h, lane, slot + S::P0 + 512);
}

// fp16 keys stay in registers.
template <int D>
struct Chunk {
    u32x4 k[2][D / 32];
    u32x4 v[D / 16];
};
template <bool PAST>
__device__ __forceinline__ u32x4 load_piece(const char* at) {
    return PAST ? __builtin_nontemporal_load((const u32x4*)at) : *(const u32x4*)at;
}
template <bool PAST, int D>
__device__ __forceinline__ void load_k(Chunk<D>& x, const PagedView& c, const Place& p, int h, int lane) {
    const char* row = k_row(c, p, h, lane, 2 * D);
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
        for (int j = 0; j < D / 32; j++) x.k[t][j] = load_piece<PAST>(row + t * 8 * D + 64 * j);
}
template <bool PAST, int D>
__device__ __forceinline__ void load_v(Chunk<D>& x, const PagedView& c, const Place& p, int h, int lane) {
    const char* at = c.v + block_of(c, p, h, lane >> 4) * (D * 16) + 16 * (lane & 15);
#pragma unroll
    for (int j = 0; j < D / 16; j++) x.v[j] = load_piece<PAST>(at + 256 * j);
}

// 8 codes of a K piece, its step e, as halves code * 2^-24.
template <int BITS>
__device__ __forceinline__ half8 k_codes(u32x4 k, int e) {
    if constexpr (BITS == 16) {
        return as_h8(k);
    } else if constexpr (BITS == 8) {
        const uint32_t w0 = k[2 * e], w1 = k[2 * e + 1];
        return as_h8(u32x4{__builtin_amdgcn_perm(0u, w0, 0x0C010C00u), __builtin_amdgcn_perm(0u, w0, 0x0C030C02u),
                           __builtin_amdgcn_perm(0u, w1, 0x0C010C00u), __builtin_amdgcn_perm(0u, w1, 0x0C030C02u)});
    } else {
        const uint32_t w = k[e], f = 0x000F000Fu;
        return as_h8(u32x4{w & f, w >> 4 & f, w >> 8 & f, w >> 12 & f});
    }
}
// 8 keys' codes of dim e of a V piece; of 4 bits pairs 1 and 3 at 16 times their value.
template <int BITS>
__device__ __forceinline__ half8 v_codes(u32x4 v, int e) {
    if constexpr (BITS == 16) {
        return as_h8(v);
    } else if constexpr (BITS == 8) {
        const uint32_t w0 = v[2 * e], w1 = v[2 * e + 1];
        return as_h8(u32x4{__builtin_amdgcn_perm(0u, w0, 0x0C010C00u), __builtin_amdgcn_perm(0u, w0, 0x0C030C02u),
                           __builtin_amdgcn_perm(0u, w1, 0x0C010C00u), __builtin_amdgcn_perm(0u, w1, 0x0C030C02u)});
    } else {
        const uint32_t w = v[e], w8 = w >> 8;
        return as_h8(u32x4{w & 0x000F000Fu, w & 0x00F000F0u, w8 & 0x000F000Fu, w8 & 0x00F000F0u});
    }
}

// The codes' middle, negative, 8 times (of 4 bits as v_codes holds the pairs), or zeros.
template <int BITS>
__device__ __forceinline__ half8 middle(bool here) {
    const uint32_t a = here ? (BITS == 4 ? 0xC800C800u : 0xD800D800u) : 0u, b = BITS == 4 ? (here ? 0xD800D800u : 0u) : a;
    return as_h8(u32x4{a, b, a, b});
}

// The same number, of which the compiler keeps nothing from one use to the next: what is formed of it costs a few
// instructions each time, where kept in registers it drove others to memory.
__device__ __forceinline__ int afresh(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

__device__ __forceinline__ float4v mfma(half8 a, half8 b, float4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Columns of a piece's rows that are joined over LDS at a time.
constexpr int kJoin = 128;
// Floats of LDS that hold the waves' keys, or their rows being joined [WAVES][rows][kJoin + 4].
template <int BITS, int D, bool INT8, int TILES>
__host__ __device__ constexpr int key_floats(int rows) {
    const int waves = Form<BITS, D, TILES>::WAVES;
    const int join = waves * rows * (kJoin + 4), keys = Form<BITS, D, TILES>::RING ? waves * Shape<BITS, D, INT8>::SLOT / 4 : 0;
    return join > keys ? join : keys;
}

template <int BITS, int D, bool INT8, int TILES, bool PAST>
__global__ __launch_bounds__((64 * Form<BITS, D, TILES>::WAVES), (Form<BITS, D, TILES>::SIMD)) void paged_attend_kernel(AttendArgs a) {
    using C = Shape<BITS, D, INT8>;
    using F = Form<BITS, D, TILES>;
    constexpr bool RING = F::RING;
    constexpr int RT = TILES, KW = F::WAVES, NT = 64 * KW;
    constexpr int NG = C::NG, STEPS = D / 32, DPP = C::DPP, QS = D + 8, PPS = 16 / BITS;  // K steps of a piece
    extern __shared__ __attribute__((aligned(16))) float lds[];  // keys or joins, (max, sum) [TILES][KW][16], q [rows][QS]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), h = blockIdx.y;
    const int col = lane & 15, g = lane >> 4;
    const int row0 = (int)blockIdx.z * TILES * 16;  // the workgroup's first
    const int tile_rows = min(a.R - row0, 16);      // of the first tile
    const int q_rows = TILES == 1 ? tile_rows : 16 * TILES, q_col = TILES == 1 ? min(col, tile_rows - 1) : col;
    float2* sml = (float2*)(lds + key_floats<BITS, D, INT8, TILES>(tile_rows));
    f16* sq = (f16*)(sml + TILES * KW * 16);

    const uint32_t w = blockIdx.x;
    uint32_t at = 0, end = 0, per, rest, total;  // (one piece: end stays below)
    Piece piece;
    auto zeros = [&](int b) {  // of a sequence without keys
        const int64_t at = (b * (int64_t)a.c.hkv + h) * a.R + row0;
        for (int i = threadIdx.x; i < min(a.R - row0, 16 * RT) * (D / 4); i += NT) *(half4v*)(a.out + at * D + 4 * i) = half4v{};
    };
    auto whole_from = [&](int b) {
        for (; b < a.n_seq; b += gridDim.x) {
            const int len = min(max(a.lengths[b], 0), a.width << a.c.lg);
            const uint32_t all = (uint32_t)(keys_of(a, len) + a.round - 1) / a.round;
            if (all) return Piece{b, len, 0, all, all, 0};
            zeros(b);
        }
        return Piece{-1, 0, 0, 0, 0, 0};
    };
    if (a.whole) {
        per = rest = total = 0;
        piece = whole_from(w);
    } else {
        const Plan plan = plan_of(a);
        per = plan.per, rest = plan.rest, total = plan.total;
        if (a.n_seq > 64) {  // (else the second launch's)
            for (int b0 = 64 * w; b0 < a.n_seq; b0 += 64 * gridDim.x) {
                const uint32_t n = b0 + lane < a.n_seq ? rounds_of(a, b0 + lane) : 1u;
                for (uint64_t none = __ballot(n == 0); none; none &= none - 1) zeros(b0 + __builtin_ctzll(none));
            }
            if ((threadIdx.x | h | row0) == 0) a.cut[w].x = ~0u;
        }
        if (!plan.most) {
            if (w >= plan.workers) return;
            at = w * per + min(w, rest);
            end = at + per + (w < rest);
        }
        piece = first_piece(a, plan, w, at);
    }
    for (bool first = true; piece.b >= 0; first = false) {
        const int b = piece.b, len = piece.len, keys = keys_of(a, len);
        const uint32_t r0 = piece.r0, r1 = piece.r1;
        const int32_t* table = a.table + b * a.table_stride;
        const int32_t* picked = a.picked ? a.picked + ((int64_t)b * a.c.hkv + h) * a.n_picked : nullptr;
        Places ahead;
        auto look = [&](uint32_t r) {
            const int ln = afresh(lane);
            const int64_t key = (int64_t)(r + (ln >> 1)) * F::ROUND + 32 * wave + 16 * (ln & 1);
            const int j = (int)(key >> a.c.lg);
            int logical = key < keys ? (picked ? picked[j] : j) : -1;
            const int page = (uint32_t)logical < (uint32_t)a.width ? table[logical] : -1;
            const bool there = (uint32_t)page < (uint32_t)a.c.n_pages;
            ahead.page = there ? page : 0;
            ahead.pos = there ? (logical << a.c.lg) + (int)(key & ((1 << a.c.lg) - 1)) : kNoKey;
        };
        auto place_of = [&](uint32_t r) {
            Place p{};
            if (r >= r1) return p;  // (behind the piece: not requested)
            const int i = (int)((r - r0) & 31) * 2;
            if (i == 0) look(r);
            p.page0 = __builtin_amdgcn_readlane(ahead.page, i);
            p.page1 = __builtin_amdgcn_readlane(ahead.page, i + 1);
            p.pos0 = __builtin_amdgcn_readlane(ahead.pos, i);
            p.pos1 = __builtin_amdgcn_readlane(ahead.pos, i + 1);
            const int key = (int)(r * F::ROUND) + 32 * wave, last = (1 << a.c.lg) - 1;
            p.slot0 = key & last;
            p.slot1 = (key + 16) & last;
            return p;
        };

        Chunk<D> x;  // (not RING)
        char* slot = (char*)lds + wave * C::SLOT;
        const uint32_t slot0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)slot;
        // the query rows: requested, with the first pages, before the keys, behind which they would wait
        constexpr int QN = TILES * 16 * (D / 8) / NT;
        half8 qr[QN];
        const int tid = afresh(threadIdx.x);
#pragma unroll
        for (int i = 0; i < QN; i++) {
            const int c = (tid + NT * i) / (D / 8), d = tid % (D / 8) * 8, row = min(row0 + c, a.R - 1);
            const f16* from = a.q + b * a.q_seq + (int64_t)(h * a.G + row / a.n_rows) * a.q_head + row % a.n_rows * a.q_row;
            if (c < q_rows) qr[i] = *(const half8*)(from + d);
        }
        Place cur = place_of(r0), next{};
        if (!first) __syncthreads();  // (the last piece's rows and sums are read)
#pragma unroll
        for (int i = 0; i < QN; i++) {
            const int c = (tid + NT * i) / (D / 8), d = tid % (D / 8) * 8;
            if (c < q_rows) *(half8*)(sq + c * QS + d) = qr[i];
        }
        if constexpr (RING) {
            request_k<BITS, D, INT8, PAST>(a.c, cur, h, afresh(lane), slot0);
            request_v<BITS, D, INT8, PAST>(a.c, cur, h, afresh(lane), slot0);
        } else {
            load_k<PAST>(x, a.c, cur, h, afresh(lane));
            load_v<PAST>(x, a.c, cur, h, afresh(lane));
        }
        __syncthreads();
        float qsum[RT][NG];
        int seen[RT];  // keys before it are the row's
#pragma unroll
        for (int t = 0; t < RT; t++) {
            seen[t] = len - a.n_rows + min(row0 + 16 * t + col, a.R - 1) % a.n_rows + 1;
            if constexpr (BITS != 16) {
#pragma unroll
                for (int m = 0; m < NG; m++) {
                    // ones times q: a row's sum in every lane that holds it
                    float4v y = {0, 0, 0, 0};
#pragma unroll
                    for (int j = 0; j < STEPS / NG; j++) {
                        const half8 q = *(const half8*)(sq + (16 * t + q_col) * QS + 32 * (m * (STEPS / NG) + j) + 8 * g);
                        y = mfma(half8{} + (f16)1.0f, q, y);
                    }
                    qsum[t][m] = y[0] * (INT8 ? -128.0f * 0x1p-24f : 0x1p-24f);  // in the codes' units
                }
            }
        }
        const float sc = a.scale2 * (BITS == 16 ? 1.0f : 0x1p24f);
        const int seen_all = len - a.n_rows + 1;  // keys before it are all rows'

        float4v o[RT][D / 16], ob[RT];  // ob: the biases' part, group m's in row m
        float M[RT], l[RT];
        // V's steps so far are below 2^(E + 1) = step_end. P gives way by 2^E, so that P times the largest step takes a half's middle
        // range and lesser products keep their bits; P that meets the middles (C0 the middle code) gives way where E > 0 alone,
        // and the middles are lifted by as much instead: E is such that they then stay below 2^15. (10240 keys of 1e-3, each
        // of 2^-19 of the first one's weight, 8 bits: with no E below 0 their values' differences were lost. 17 sequences of
        // up to 8k 4-bit keys 32.4 us without, 33.3 so; Int8 the same.)
        constexpr float C0 = BITS == 4 ? 8.0f : 128.0f;
        int E = BITS == 16 ? 0 : -15;
        float step_end = 0x1p-14f, drop = 0x1p-15f;
        f16 lift = (f16)0x1p15f;
#pragma unroll
        for (int t = 0; t < RT; t++) {
            M[t] = kNone, l[t] = 0.0f;
            ob[t] = float4v{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < D / 16; i++) o[t][i] = float4v{0, 0, 0, 0};
        }
        for (uint32_t r = r0; r < r1; r++) {
            next = place_of(r + 1);
            if constexpr (RING) wait_loads<C::V_LOADS>();
            const f16* kpar = (const f16*)(slot + C::P0) + g * C::PAR;
            const int top = max(cur.pos0, cur.pos1) + 15;
            // scores: lane group g has keys 8 g + 4 u + i
            float s[RT][8];
            constexpr int QG = BITS == 16 ? 1 : NG, PER_G = STEPS / QG;
#pragma unroll
            for (int m = 0; m < QG; m++) {
                float4v acc[2][RT];
#pragma unroll
                for (int v = 0; v < 2; v++)
#pragma unroll
                    for (int t = 0; t < RT; t++) acc[v][t] = float4v{0, 0, 0, 0};
#pragma unroll
                for (int j = m * PER_G; j < (m + 1) * PER_G; j++) {
                    half8 q[RT];
#pragma unroll
                    for (int t = 0; t < RT; t++) q[t] = *(const half8*)(sq + (16 * t + q_col) * QS + 32 * j + 8 * g);
#pragma unroll
                    for (int v = 0; v < 2; v++) {
                        half8 k;
                        if constexpr (RING)
                            k = k_codes<BITS>(*(const u32x4*)(slot + (v * C::NK + j / PPS) * 1024 + 16 * lane), j % PPS);
                        else
                            k = k_codes<BITS>(x.k[v][j], 0);
#pragma unroll
                        for (int t = 0; t < RT; t++) acc[v][t] = mfma(k, q[t], acc[v][t]);
                    }
                }
                half8 ks, kb;
                if constexpr (BITS != 16) {
                    ks = *(const half8*)(kpar + 8 * m);
                    if (!INT8) kb = *(const half8*)(kpar + 8 * (NG + m));
                }
#pragma unroll
                for (int t = 0; t < RT; t++)
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float y = acc[i / 4][t][i % 4];
                        if constexpr (BITS == 16) {
                            s[t][i] = y;
                        } else if constexpr (INT8) {
                            s[t][i] = (float)ks[i] * (y + qsum[t][0]);
                        } else {
                            s[t][i] = __builtin_fmaf((float)ks[i], y, m ? s[t][i] : 0.0f);
                            s[t][i] = __builtin_fmaf((float)kb[i], qsum[t][m], s[t][i]);
                        }
                    }
                // (formed here: put off behind a branch, the compiler's choice, they keep four times as many registers)
                if constexpr (BITS != 16) {
#pragma unroll
                    for (int t = 0; t < RT; t++)
#pragma unroll
                        for (int i = 0; i < 8; i++) asm volatile("" : "+v"(s[t][i]));
                }
                if (RT > 1 && QG > 1) __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (RING) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K is read: its place takes the next
                if (r + 1 < r1) request_k<BITS, D, INT8, PAST>(a.c, next, h, afresh(lane), slot0);
            } else {
                if (r + 1 < r1) load_k<PAST>(x, a.c, next, h, afresh(lane));
            }
            __builtin_amdgcn_sched_barrier(0);
            const bool masked = top >= seen_all;
            const int pos = (g & 2 ? cur.pos1 : cur.pos0) + 8 * (g & 1);
            if constexpr (RING) {
                if (r + 1 < r1)
                    wait_loads<C::K_LOADS>();
                else
                    wait_loads<0>();
            }
            if (masked) {  // what stands behind the sequence's end takes no part, whatever it is: zeros in place of V or its scales
                constexpr int LPB = BITS == 16 ? 16 : C::PAR / 8;  // lanes of 8 keys
                const int ln = afresh(lane), blk = ln / LPB, at = (blk & 2 ? cur.pos1 : cur.pos0) + 8 * (blk & 1);
                u32x4 km;
#pragma unroll
                for (int j = 0; j < 4; j++) km[j] = (at + 2 * j < len ? 0xFFFFu : 0u) | (at + 2 * j + 1 < len ? 0xFFFF0000u : 0u);
                if constexpr (BITS != 16) {
                    u32x4* v = (u32x4*)(slot + C::P0 + 512) + ln;
                    if (ln < 4 * LPB) *v &= km;
                } else {
#pragma unroll
                    for (int j = 0; j < C::NV; j++) {
                        if constexpr (RING)
                            *((u32x4*)(slot + C::V0 + j * 1024) + ln) &= km;
                        else
                            x.v[j] &= km;
                    }
                }
            }
            const f16* vpar = kpar + 256;
            auto v_scales = [&](const f16* par, int m) { return *(const half8*)(par + 8 * m); };  // of 8 keys in group m
            // two keys' steps and bases of a group: a lane group's 16 lanes have all that there are of its 8 keys
            half2v step{}, base{};
            if constexpr (BITS != 16) {
                const int c = afresh(col);
                const f16* two = vpar + 8 * (c >> 2 & (NG - 1)) + 2 * (c & 3);
                step = *(const half2v*)two;
                if (!INT8) base = *(const half2v*)(two + 8 * NG);
            }
            float mx[RT];
#pragma unroll
            for (int t = 0; t < RT; t++) {
#pragma unroll
                for (int i = 0; i < 8; i++) s[t][i] *= sc;
                if (masked) {
#pragma unroll
                    for (int i = 0; i < 8; i++) s[t][i] = pos + i < seen[t] ? s[t][i] : -INFINITY;
                }
                mx[t] = fmaxf(fmaxf(fmaxf(s[t][0], s[t][1]), fmaxf(s[t][2], s[t][3])),
                              fmaxf(fmaxf(s[t][4], s[t][5]), fmaxf(s[t][6], s[t][7])));
            }
            float down = 1.0f;
            bool moved = false;
            if constexpr (BITS != 16) {
                half2v most = __builtin_elementwise_max(step, -step);
                if constexpr (!INT8) {
                    const half2v mid = __builtin_elementwise_fma(step, half2v{} + (f16)C0, base) * (half2v{} + (f16)0x1p-14f);
                    most = __builtin_elementwise_max(most, __builtin_elementwise_max(mid, -mid));
                }
                const float big = (float)__builtin_elementwise_max(most[0], most[1]);
                if (__any(!(big < step_end))) {
                    const int e = min(__builtin_amdgcn_readfirstlane((int)(__float_as_uint(wave_reduce(big, OpMax())) >> 23)) - 127, 16);
                    if (e > E) {
                        down = __builtin_amdgcn_exp2f((float)(E - e));
                        moved = true;
                        E = e;
                        step_end = __builtin_amdgcn_exp2f((float)(E + 1));
                        drop = __builtin_amdgcn_exp2f((float)min(E, 0));
                        lift = (f16)__builtin_amdgcn_exp2f((float)-min(E, 0));
                    }
                }
                vpar += afresh(0);  // (read again below, not held)
            }
#pragma unroll
            for (int t = 0; t < RT; t++) {
                if (__any(moved || mx[t] > M[t] + kLazy)) {
                    mx[t] = fmaxf(mx[t], lane_xor<16>(mx[t], lane));
                    mx[t] = fmaxf(mx[t], lane_xor<32>(mx[t], lane));
                    const float m1 = fmaxf(M[t], mx[t]), alpha = __builtin_amdgcn_exp2f(M[t] - m1) * down;
                    M[t] = m1;
                    l[t] *= alpha;
                    ob[t] *= alpha;
#pragma unroll
                    for (int i = 0; i < D / 16; i++) o[t][i] *= alpha;
                }
                const float ref = M[t] + ((float)E - kLift);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    s[t][i] = __builtin_amdgcn_exp2f(s[t][i] - ref);
                    l[t] += s[t][i];
                }
            }
            half8 ph[RT];
            if constexpr (BITS == 16 || !INT8) {
#pragma unroll
                for (int t = 0; t < RT; t++)
#pragma unroll
                    for (int i = 0; i < 8; i++) ph[t][i] = BITS == 16 ? (f16)s[t][i] : (f16)__builtin_fmaf(s[t][i], drop, 0.0f);
            }
            if constexpr (BITS == 16) {
#pragma unroll
                for (int j = 0; j < C::NV; j++) {
                    u32x4 v;
                    if constexpr (RING)
                        v = *(const u32x4*)(slot + C::V0 + j * 1024 + 16 * lane);
                    else
                        v = x.v[j];
#pragma unroll
                    for (int t = 0; t < RT; t++) o[t][j] = mfma(as_h8(v), ph[t], o[t][j]);
                }
            } else {
                if constexpr (!INT8) {
                    half8 vb = __builtin_elementwise_fma(v_scales(vpar, min(col, NG - 1)), half8{} + (f16)C0, v_scales(vpar, NG + min(col, NG - 1))) * lift;
                    if (col >= NG) vb = half8{};
#pragma unroll
                    for (int t = 0; t < RT; t++) ob[t] = mfma(vb, ph[t], ob[t]);
                }
                if constexpr (BITS == 4) {
#pragma unroll
                    for (int t = 0; t < RT; t++)
                        s[t][2] *= 0.0625f, s[t][3] *= 0.0625f, s[t][6] *= 0.0625f, s[t][7] *= 0.0625f;
                }
                constexpr int PER = C::NV / NG;
#pragma unroll
                for (int m = 0; m < NG; m++) {
                    const half8 vs = v_scales(vpar, m);
#pragma unroll
                    for (int t = 0; t < RT; t++) {
#pragma unroll
                        for (int i = 0; i < 8; i++) ph[t][i] = (f16)__builtin_fmaf(s[t][i], (float)vs[i], 0.0f);
                        ob[t] = mfma(middle<BITS>(afresh(col) == m), ph[t], ob[t]);
                    }
#pragma unroll
                    for (int j = m * PER; j < (m + 1) * PER; j++) {
                        const u32x4 piece = *(const u32x4*)(slot + C::V0 + j * 1024 + 16 * lane);
#pragma unroll
                        for (int e = 0; e < DPP; e++) {
                            const half8 v = v_codes<BITS>(piece, e);
#pragma unroll
                            for (int t = 0; t < RT; t++) o[t][j * DPP + e] = mfma(v, ph[t], o[t][j * DPP + e]);
                        }
                    }
                    if (RT > 1) __builtin_amdgcn_sched_barrier(0);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (RING) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                if (r + 1 < r1) request_v<BITS, D, INT8, PAST>(a.c, next, h, afresh(lane), slot0);
            } else {
                if (r + 1 < r1) load_v<PAST>(x, a.c, next, h, afresh(lane));
            }
            __builtin_amdgcn_sched_barrier(0);
            cur = next;
        }
        if constexpr (RING) __syncthreads();  // (every wave has read its keys: their place takes the rows)

        // the rows' sums over the lane groups, biases, and the waves of a tile joined
        const bool done = r0 == 0 && r1 == piece.all;
#pragma unroll
        for (int t = 0; t < RT; t++) {
            l[t] += lane_xor<16>(l[t], lane);
            l[t] += lane_xor<32>(l[t], lane);
            if (g == 0) sml[(t * KW + wave) * 16 + col] = float2{M[t] + (float)E, l[t]};
        }
        float* so = lds + (wave * tile_rows + col) * (kJoin + 4);
#pragma unroll
        for (int t = 0; t < RT; t++) {
            const int rows = min(a.R - row0 - 16 * t, 16);  // (none or fewer: nothing is written)
            float bias[NG];
#pragma unroll
            for (int m = 0; m < NG; m++)
                bias[m] = BITS == 16 ? 0.0f : __shfl(ob[t][m & 3], col);
#pragma unroll
            for (int part = 0; part < D / kJoin; part++) {
                constexpr int PJ = C::NV * kJoin / D;  // V pieces of a part
                if (t > 0 || part > 0) __syncthreads();  // (the last part is read)
                if (col < rows) {
#pragma unroll
                    for (int jj = 0; jj < PJ; jj++) {
                        const int j = part * PJ + jj;
                        float f[4 * DPP];  // dims DPP (16 jj + 4 g) .. of the part
#pragma unroll
                        for (int i = 0; i < 4; i++)
#pragma unroll
                            for (int e = 0; e < DPP; e++) {
                                const float y = o[t][j * DPP + e][i];
                                f[i * DPP + e] = BITS == 16 ? y : __builtin_fmaf(y, 0x1p24f, bias[INT8 ? 0 : j / (C::NV / NG)]);
                            }
#pragma unroll
                        for (int i = 0; i < DPP; i++)
                            *(float4v*)(so + DPP * (16 * jj + 4 * g) + 4 * i) = float4v{f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]};
                    }
                }
                __syncthreads();
                for (int i = afresh(threadIdx.x); i < rows * (kJoin / 4); i += NT) {
                    const int c = i / (kJoin / 4), d = i % (kJoin / 4) * 4;
                    float mm = kNone;
#pragma unroll
                    for (int k = 0; k < KW; k++) mm = fmaxf(mm, sml[(t * KW + k) * 16 + c].x);
                    float4v y = {0, 0, 0, 0};
                    float sum = 0.0f;
#pragma unroll
                    for (int k = 0; k < KW; k++) {
                        const float2 ml = sml[(t * KW + k) * 16 + c];
                        const float f = __builtin_amdgcn_exp2f(ml.x - mm);
                        y += f * *(const float4v*)(lds + (k * tile_rows + c) * (kJoin + 4) + d);
                        sum = __builtin_fmaf(f, ml.y, sum);
                    }
                    const int64_t rw = row0 + 16 * t + c;
                    if (done) {
                        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                        const int64_t to = ((b * (int64_t)a.c.hkv + h) * a.R + rw) * D + part * kJoin + d;
                        *(half4v*)(a.out + to) = half4v{(f16)(y[0] * inv), (f16)(y[1] * inv), (f16)(y[2] * inv), (f16)(y[3] * inv)};
                    } else {
                        const int64_t to = ((int64_t)piece.slot * a.c.hkv + h) * a.R + rw;
                        *(float4v*)(a.part_o + to * D + part * kJoin + d) = y;
                        if (part == 0 && d == 0) a.part_ml[to] = float2{mm, sum};
                    }
                }
            }
        }
        if (a.whole) {
            piece = whole_from(b + gridDim.x);
            continue;
        }
        if (a.n_seq > 64 && r0 == 0 && r1 < piece.all && (threadIdx.x | h | row0) == 0)
            a.cut[w] = uint4{(uint32_t)b, at, piece.all, total};
        at += r1 - r0;
        if (at >= end) return;
        piece = piece_from(a, per, rest, w, at, b + 1, at);
    }
}

// Joins a row's pieces: grid (rows of all heads, n_seq). A sequence within one worker's run was written
// by it; one without keys is zeros. Above 64 sequences grid (rows of all heads, workers): a worker's part of
// it is the sequence that its run leaves unfinished, if it begins there (by sequences, each looking for its place: 1024 of up
// to 256 keys, D = 128, 8 bits, 297 us for 130).
template <int D>
__global__ __launch_bounds__(256) void paged_merge_kernel(AttendArgs a) {
    constexpr int TC = D / 4, SG = 256 / TC;
    __shared__ float4v sm_o[256];
    __shared__ float sm_l[SG];
    const int tid = threadIdx.x, h = (int)blockIdx.x / a.R, row = (int)blockIdx.x % a.R;
    const int lane = tid & 63;
    int b = blockIdx.y;
    Plan plan;
    uint32_t mine, before; // the sequence's rounds, and those before it
    if (a.cut) {
        const uint4 x = a.cut[b];
        b = (int)x.x;
        if (b < 0) return;
        before = x.y, mine = x.z;
        plan.workers = min((uint32_t)a.workers, x.w);
        plan.per = x.w / plan.workers;
        plan.rest = x.w - plan.per * plan.workers;
        plan.most = 0;
    } else {
        plan = plan_of(a);  // (above 64: tables without columns)
        mine = a.n_seq > 64 ? 0u : (uint32_t)__builtin_amdgcn_readlane((int)plan.rounds, b);
        before = a.n_seq > 64 ? 0u : (uint32_t)__builtin_amdgcn_readlane((int)plan.through, b) - mine;
    }
    uint32_t n, slot0;  // its pieces, the first one's slot
    int64_t step;
    const int d = tid % TC * 4, sg = tid / TC;
    f16* to = a.out + ((b * (int64_t)a.c.hkv + h) * a.R + row) * D + d;
    if (mine == 0) {
        if (sg == 0) *(half4v*)to = half4v{};
        return;
    }
    if (plan.most) {
        n = (uint32_t)__builtin_amdgcn_readlane((int)plan.pieces, b);
        slot0 = 2 * ((uint32_t)__builtin_amdgcn_readlane((int)plan.last, b) - n);
        step = slot0;
    } else {
        // the worker of a round, and where its run begins; a sequence's first piece is the last of its worker's run,
        // unless that begins with it
        const uint32_t longer = plan.rest * (plan.per + 1);
        auto worker_of = [&](uint32_t x) {
            return x < longer ? x / (plan.per + 1) : plan.rest + (x - longer) / plan.per;
        };
        const uint32_t w0 = worker_of(before), w1 = worker_of(before + mine - 1);
        n = w1 - w0 + 1;
        slot0 = w0 * plan.per + min(w0, plan.rest) == before ? 2 * w0 : 2 * w0 + 1;
        step = 2 * w0;
    }
    if (n == 1) return;
    auto slot_of = [&](uint32_t i) { return ((int64_t)(i == 0 ? slot0 : step + 2 * i) * a.c.hkv + h) * a.R + row; };
    float mm = kNone;
    for (uint32_t i = lane; i < n; i += 64) mm = fmaxf(mm, a.part_ml[slot_of(i)].x);
    mm = wave_reduce(mm, OpMax());
    float4v y = {0, 0, 0, 0};
    float sum = 0.0f;
    constexpr int AHEAD = 8;  // pieces in flight
    for (uint32_t i = sg; i < n; i += SG * AHEAD) {
        float2 ml[AHEAD];
        float4v x[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; k++) {
            const int64_t s = slot_of(min(i + k * SG, n - 1));
            ml[k] = a.part_ml[s];
            x[k] = *(const float4v*)(a.part_o + s * D + d);
        }
#pragma unroll
        for (int k = 0; k < AHEAD; k++) {
            const float f = i + k * SG < n ? __builtin_amdgcn_exp2f(ml[k].x - mm) : 0.0f;
            y += f * x[k];
            sum = __builtin_fmaf(f, ml[k].y, sum);
        }
    }
    sm_o[tid] = y;
    if (tid % TC == 0) sm_l[sg] = sum;
    __syncthreads();
    if (sg) return;
#pragma unroll
    for (int k = 1; k < SG; k++) {
        y += sm_o[k * TC + tid];
        sum += sm_l[k];
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    *(half4v*)to = half4v{(f16)(y[0] * inv), (f16)(y[1] * inv), (f16)(y[2] * inv), (f16)(y[3] * inv)};
}

template <int BITS, int D, bool INT8, int TILES>
size_t attend_lds(int R) {
    const int rows = std::min(R, 16), q_rows = TILES == 1 ? rows : 16 * TILES;
    return (size_t)key_floats<BITS, D, INT8, TILES>(rows) * 4 + TILES * Form<BITS, D, TILES>::WAVES * 16 * 8 + (size_t)q_rows * (D + 8) * 2;
}
template <int BITS, int D, bool INT8, int TILES, bool PAST>
int launch_attend(const AttendArgs& a, hipStream_t stream) {
    const size_t lds = attend_lds<BITS, D, INT8, TILES>(a.R);
    static_assert(BITS == 16 || 8 * Shape<BITS, D, INT8>::PAR <= 512, "K's and V's scales and biases of 32 keys have 512 bytes each");
    const void* f = (const void*)paged_attend_kernel<BITS, D, INT8, TILES, PAST>;
    if (int rc = ensure_dynamic_lds(f, lds)) return rc;
    const dim3 grid(a.workers, a.c.hkv, (a.R + 16 * TILES - 1) / (16 * TILES));
    hipLaunchKernelGGL((paged_attend_kernel<BITS, D, INT8, TILES, PAST>), grid, dim3(64 * Form<BITS, D, TILES>::WAVES), lds, stream, a);
    QW_HIP_CHECK(hipGetLastError());
    return QW_OK;
}
template <class F>
int by_shape(int bits, bool int8, int D, int n_tiles, F f) {
    using std::integral_constant;
    auto tiles = [&](auto b, auto i8, auto d) {
        return n_tiles == 1 ? f(b, i8, d, integral_constant<int, 1>()) : f(b, i8, d, integral_constant<int, 2>());
    };
    auto dims = [&](auto b, auto i8) {
        return D == 256 ? tiles(b, i8, integral_constant<int, 256>()) : tiles(b, i8, integral_constant<int, 128>());
    };
    if (bits == 16) return dims(integral_constant<int, 16>(), integral_constant<bool, false>());
    if (bits == 4) return dims(integral_constant<int, 4>(), integral_constant<bool, false>());
    if (int8) return dims(integral_constant<int, 8>(), integral_constant<bool, true>());
    return dims(integral_constant<int, 8>(), integral_constant<bool, false>());
}

}  // namespace

int check_query(const PagedCache& c, const PagedQuery& q, const char* what) {
    const std::string w(what);
    QW_REQUIRE(q.n_seq >= 0 && q.n_seq <= 65535 && q.n_rows > 0 && q.n_q_heads > 0 && q.n_q_heads % c.hkv == 0,
               QW_ERR_INVALID_ARGUMENT, w + ": 0 .. 65535 sequences, n_rows > 0 and n_q_heads a multiple of the KV heads expected");
    QW_REQUIRE(q.n_seq == 0 || (q.q && q.lengths && (q.table || q.table_width == 0)), QW_ERR_INVALID_ARGUMENT, w + ": null q/lengths/table");
    QW_REQUIRE(q.table_width >= 0 && q.table_stride >= q.table_width && (int64_t)q.table_width * c.page_size <= 0x7fffff00,
               QW_ERR_INVALID_ARGUMENT, w + ": table_width >= 0, not above its stride, and table_width * page_size < 2^31 expected");
    QW_REQUIRE((uintptr_t)q.q % 16 == 0 && (q.seq_stride | q.head_stride | q.row_stride) % 8 == 0 && q.seq_stride >= 0 &&
                   q.head_stride >= 0 && q.row_stride >= 0,
               QW_ERR_INVALID_ARGUMENT, w + ": q 16-byte aligned with strides of whole 16 bytes expected");
    const int64_t rows = (int64_t)(q.n_q_heads / c.hkv) * q.n_rows;
    QW_REQUIRE(rows <= 16384 && rows * c.hkv <= (1 << 22), QW_ERR_UNSUPPORTED, w + ": at most 16384 query rows a KV head");
    return QW_OK;
}

int paged_attention(PagedCache& c, const PagedQuery& q, const int32_t* picked, int n_picked, float scale, void* out,
                    hipStream_t stream) {
    if (int rc = check_query(c, q, "paged attention")) return rc;
    QW_REQUIRE(scale >= -0x1p40f && scale <= 0x1p40f, QW_ERR_INVALID_ARGUMENT, "paged attention: |scale| <= 2^40 expected");
    QW_REQUIRE(!picked || (n_picked > 0 && (int64_t)n_picked * c.page_size <= 0x7fffff00), QW_ERR_INVALID_ARGUMENT,
               "paged attention: n_picked > 0 with n_picked * page_size < 2^31 expected");
    if (q.n_seq == 0) return QW_OK;
    QW_REQUIRE(out && (uintptr_t)out % 8 == 0, QW_ERR_INVALID_ARGUMENT, "paged attention: out null or off 8 bytes");
    const int64_t most = std::min<int64_t>(q.table_width, picked ? n_picked : q.table_width) * c.page_size;  // keys of a sequence
    // Two row tiles a workgroup, which takes a key once for both, above 16 rows. One / two, 4 sequences over 16k keys, us: 18 rows,
    // D = 256, Int8 45.9 / 37.2, 4 bits 38.4 / 35.9, fp16 83.4 / 53.8; 20 rows, D = 128, 8 bits 50.0 / 36.6, fp16 84.4 / 51.5;
    // 72 rows, D = 256, Int8 89.4 / 62.1.
    const int tiles = (q.n_q_heads / c.hkv) * q.n_rows <= 16 ? 1 : 2;
    // as many workers as the card holds at a time, all heads and row tiles counted
    int held = 0, round = 0;
    by_shape(c.bits, c.int8(), c.D, tiles, [&](auto b, auto i8, auto d, auto t) {
        using F = Form<decltype(b)::value, decltype(d)::value, decltype(t)::value>;
        const size_t lds = attend_lds<decltype(b)::value, decltype(d)::value, decltype(i8)::value, decltype(t)::value>(
            (q.n_q_heads / c.hkv) * q.n_rows);
        held = std::max(1, std::min<int>(4 * F::SIMD / F::WAVES, (int)(160 * 1024 / lds)));
        round = F::ROUND;
        return QW_OK;
    });
    const int64_t rounds = (most + round - 1) / round * q.n_seq;
    QW_REQUIRE(rounds < (1ll << 31), QW_ERR_UNSUPPORTED, "paged attention: n_seq * table_width * page_size below 2^38 expected");
    // (one handle, a stream a thread: they would share a workspace)
    QW_REQUIRE(stream != hipStreamPerThread, QW_ERR_UNSUPPORTED, "paged attention: hipStreamPerThread; name a stream");
    DeviceGuard dg(c.device);
    QW_REQUIRE(dg.ok, QW_ERR_HIP, "paged attention: hipSetDevice failed");
    AttendArgs a{};
    a.c = c.view;
    a.q = (const f16*)q.q;
    a.q_seq = q.seq_stride, a.q_head = q.head_stride, a.q_row = q.row_stride;
    a.out = (f16*)out;
    a.lengths = q.lengths;
    a.table = q.table;
    a.table_stride = q.table_stride;
    a.width = q.table_width;
    a.n_seq = q.n_seq;
    a.G = q.n_q_heads / c.hkv;
    a.n_rows = q.n_rows;
    a.R = a.G * q.n_rows;
    a.picked = picked;
    a.n_picked = n_picked;
    a.scale2 = scale * kLog2e;
    const int groups = (a.R + 16 * tiles - 1) / (16 * tiles);
    a.round = round;
    a.workers = (int)std::max<int64_t>(1, std::min<int64_t>(rounds, 256 * held / ((int64_t)c.hkv * groups)));
    // A sequence of few rounds is read by one worker where the rounds one after another cost less than the second launch,
    // which joins pieces (of one round none is cut anyway). Whole / cut, a pass in us, 1 sequence: D = 256, 8 bits, 3 rounds
    // 11.7 / 12.0, 5 rounds 15.6 / 12.1, fp16 12.8 / 12.8 and 17.2 / 13.1; D = 128, 8 bits, 3 rounds 9.0 / 11.2, 5
    // rounds 11.7 / 11.2, fp16 8.0 / 11.2 and 9.9 / 11.2. 16 sequences, D = 128, 5 rounds 12.4 / 13.9 and 11.0 / 16.3. With
    // more than 64, whose cuts take a search, up to 8: D = 128, 8 bits, 65 sequences 32.0 / 34.9, 128 41.0 / 50.8, 256 97.7 /
    // 102, 1024 374 / 368; D = 256, 4 bits, 128 32.9 / 49.8, 1024 246 / 255. (8 for all: that one of them loses 2 %.)
    const int few = q.n_seq > 64 ? 8 : c.D == 256 ? 3 : c.bits == 16 ? 5 : 4;
    // (one worker, where the query rows alone fill the card, reads all of every sequence)
    a.whole = rounds > 0 && (a.workers == 1 || most <= few * round);
    // Keys that may be more than the 256 MB behind the L2 caches, each read once, go past the caches (us, without / with: 64
    // sequences of up to 16k fp16 keys 491 / 438, 32 sparse ones of 32k fp16 keys, with the selection, 127 / 112). Fewer may be there
    // from the last call (64 of up to 1024 fp16 keys, the same again and again, 44.5 / 52.1; where others came between, 200 MB
    // of 4 sequences' Int8 keys with 5 rows, 50.1 / 48.6), and more row tiles than a workgroup's share them (128 rows of 4 sequences, 8k fp16 keys, 182 / 236).
    // The host knows the lists' and tables' room and the pool's, not the lengths: sequences cannot have more keys of their own
    // than the pool, however wide their tables (64 sequences of up to 1024 fp16 keys in tables of 8192 columns 40.3 / 34.1).
    const double keys = std::min((double)most * q.n_seq, (double)c.n_pages * c.page_size);
    const bool past = groups == 1 && keys * c.hkv * (c.D * c.bits / 4 + c.par_halves() / 2) > 256.0 * (1 << 20);
    const int64_t parts = (int64_t)a.workers * 2 * c.hkv * a.R;
    const bool cuts = q.n_seq > 64 && rounds > 0 && !a.whole;
    if (!a.whole) {
        void* ws = nullptr;
        if (int rc = workspace(kWsPaged, c.device, stream, (size_t)(parts * (c.D * 4 + 8) + (cuts ? a.workers * 16 : 0)), &ws)) return rc;
        a.part_o = (float*)ws;
        a.part_ml = (float2*)(a.part_o + parts * c.D);
        a.cut = cuts ? (uint4*)(a.part_ml + parts) : nullptr;
    }
    if (rounds > 0) {
        const int rc = by_shape(c.bits, c.int8(), c.D, tiles, [&](auto b, auto i8, auto d, auto t) {
            constexpr int B = decltype(b)::value, D = decltype(d)::value, T = decltype(t)::value;
            return past ? launch_attend<B, D, decltype(i8)::value, T, true>(a, stream) : launch_attend<B, D, decltype(i8)::value, T, false>(a, stream);
        });
        if (rc) return rc;
    }
    if (a.whole) return QW_OK;
    const dim3 grid((unsigned)(c.hkv * a.R), cuts ? a.workers : q.n_seq);
    if (c.D == 256)
        hipLaunchKernelGGL(paged_merge_kernel<256>, grid, dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL(paged_merge_kernel<128>, grid, dim3(256), 0, stream, a);
    QW_HIP_CHECK(hipGetLastError());
    return QW_OK;
}

}  // namespace qw
