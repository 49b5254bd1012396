// shared_plan.hpp -- the work axis of the shared-keys kernel (shared_tile.hpp): what
// the plan kernel writes, how ranges of the axis map to workgroups and to partial
// rows.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "shared_attn.hpp"

namespace vmc {

// One set of keys and the rows that attend them.  Paged calls: the groups' common
// keys, then every row's own; contiguous calls: the sequences.
struct SetDesc {
    int row0, ntok;  // first row, rows (tokens); each stands for G query heads a KV head
    int klo, khi;    // keys klo .. khi - 1 (tiles start at klo rounded down to 16)
    int src;         // block-table row, or the key that key 0 is
    int nb;          // items a KV head: ceil(ntok * G / rows of an item)
    int tiles;       // 64-key tiles of an item
    int own;         // paged: a row's own keys (else each row has seq_lens[row] at most)
};

// Where a range begins: its first tile, and how many it has.
struct RangeRec {
    int set, g, rb, t, ntiles;
    int pad[3];
    SetDesc d;  // of the set
};

// Paged calls: what the merge needs of one row.
struct RowRec {
    int64_t own_u, grp_u;       // first unit of the set's first item
    int own_tiles;              // 0: none
    int grp_tiles, grp_nb, grp_row0, grp_ntok;
    int pad[3];
};

// An item's first kItemCost units stand for what a workgroup spends on the item beside
// its tiles (the next rows' Q, the last rows' partial results), so that a range of
// short items gets fewer tiles.  2: 64 rows over 32768 common and 32 to 2048 own tokens
// take 96.7 us, 101.5 with 1; 24 ragged targets 39.0, 38.1 with 1.
constexpr int kItemCost = 2;

constexpr int kTileWaves = 4;  // waves of the shared-keys kernel, 32 rows each
constexpr int kTileRows = 32 * kTileWaves;  // rows of an item (GGUF pages: half)
// its workgroups that fit a CU: 64 KB of tiles (head_dim 64: 48, 256: 128), 168 registers a
// lane at head_dim 64 (two workgroups there: 43 instead of 35 us, the kernel alone, for 48
// rows with 64 to 4096 tokens of their own), 256 at 128, 512 at 256
__host__ __device__ constexpr int tile_per_cu(int D) { return D == 64 ? 3 : D == 128 ? 2 : 1; }

// Sets of a call whose plan every workgroup of the shared-keys kernel makes for itself, in
// LDS (about the last size that leaves head_dim 64 its three workgroups a CU): the plan
// kernel takes 5 to 8 us, this 2 to 3.  Not for whole items, of which a CU
// takes one after the other, and each would plan again.
constexpr int kPlanFused = 96;

struct PlanParams {
    const int32_t* starts;
    const int32_t* set_lens;
    const int32_t* seq_lens;    // paged
    const int32_t* key_starts;  // contiguous
    int ns, rows;               // groups or sequences; rows
    int nsets;                  // sets: ns (+ rows where paged)
    int max_keys, num_keys;
    int Hkv, G, RB;
    int paged, whole;
    int grid, cus;    // ranges at most, CUs
    int64_t* cum;     // [nsets + 1] units (whole: items) before each set
    int64_t* cumt;    // [nsets + 1] tiles before each set
    SetDesc* desc;    // [nsets]
    RangeRec* range;  // [grid] (not whole)
    RowRec* row;      // [rows] (paged)
    int32_t* gs;      // [ns + 1] starts, cut to [0, rows] and made non-decreasing
};

struct TileParams {
    uint16_t* out;
    const uint16_t* q;
    int64_t q_ts, q_hs;
    int Hq, Hkv, G;
    float scale;
    const int64_t* cum;
    const SetDesc* desc;
    const RangeRec* range;
    const RowRec* row;
    int ns, nsets, paged, whole;
    int fused;       // the kernel makes the plan itself
    PlanParams plan;
    int total_rows;
    int grid, cus;   // ranges at most, CUs
    float* part;     // partial rows of D + 4 floats: o, m, l, two unused
    const uint8_t* kp;
    const uint8_t* vp;
    int64_t k_row, k_head, v_row, v_head;  // bytes between keys (paged: of a page; v as k), between heads
    int64_t page_bytes, max_blocks;
    int bs;
    const int32_t* bt;
    const int32_t* seq_lens;
};

int shared_tile_d64(const TileParams& p, int src, bool q_bf16, unsigned grid, hipStream_t s);
int shared_tile_d128(const TileParams& p, int src, bool q_bf16, unsigned grid, hipStream_t s);
int shared_tile_d256(const TileParams& p, int src, bool q_bf16, unsigned grid, hipStream_t s);

// The MFMA path of a call: whether it takes the shape, what workspace it needs (its
// sizes alone decide), and the launches.
bool shared_tiles_take(const SharedArgs& a);
size_t shared_tiles_workspace(bool paged, int rows, int nsets, int Hq, int Hkv, int D);
int shared_tiles(const SharedArgs& a, void* ws, hipStream_t s);

namespace {

// Ranges that a total of units is cut into: a range a CU from single units, more from
// kUnitsMin units each on, the grid at most.  Four rows over 512 tokens (200 units): 13.2
// us, 16.6 with kUnitsMin each; 16 rows over 4096 tokens of q8_0 (1104 units): 21.8
// us, 22.7 with fewer each.
constexpr int kUnitsMin = kItemCost + 1;  // one tile of an item

__host__ __device__ __forceinline__ int plan_ranges(int64_t total, int grid, int cus) {
    int64_t n = (total + kUnitsMin - 1) / kUnitsMin;
    const int64_t few = total < cus ? total : cus;
    n = n > few ? n : few;
    return (int)(n < grid ? n : grid);
}

// the range that holds unit u of total, ranges w being [w total / n, (w + 1) total / n)
__device__ __forceinline__ int plan_range_of(int64_t u, int64_t total, int n) {
    const int64_t x = (u + 1) * n - 1;
    if (((x | total) >> 32) == 0) return (int)((uint32_t)x / (uint32_t)total);
    return (int)(x / total);
}

// last s in [0, n) with cum[s] <= u (cum non-decreasing, cum[0] <= u); one wave, 64
// probes a round
template <typename T>
__device__ __forceinline__ int plan_find(const T* cum, int n, int64_t u, int lane) {
    int lo = 0, len = n;
    while (len > 1) {
        const int step = (len + 63) / 64;
        const int64_t at = (int64_t)lane * step;
        const bool in = at < len && (int64_t)cum[lo + (at < len ? at : 0)] <= u;
        const int k = __popcll(__ballot(in)) - 1;
        lo += max(k, 0) * step;
        len = min(step, len - max(k, 0) * step);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

// First partial row of the piece of item (g, rb) of set d in a range.  Pieces follow
// the axis, where each step goes to the next item or the next range: range *
// rb_rows + (rows of the items before) grows by at least a piece's rows with
// each step.  grid * rb_rows + 2 * rows * Hq rows in all.
__device__ __forceinline__ int64_t plan_rows_paged(int range, int rb_rows, int Hq, int G, int rows, int own, int row0,
                                                   int ntok, int g, int rb) {
    return (int64_t)range * rb_rows + (int64_t)Hq * ((own ? rows : 0) + (int64_t)row0) + (int64_t)g * ntok * G +
           rb * rb_rows;
}

// Contiguous calls write whole items directly: a range has two cut ones at most, one
// that began before it and one that goes on behind it
__device__ __forceinline__ int64_t plan_rows_local(int range, int rb_rows, bool began_before) {
    return (2 * (int64_t)range + (began_before ? 0 : 1)) * rb_rows;
}

}  // namespace
}  // namespace vmc
