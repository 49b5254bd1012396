// shared_plan_dev.hpp -- the steps of the plan (shared_plan.hpp) as device code, for
// the plan kernels and for the shared-keys kernel's own start.
#pragma once

#include "shared_plan.hpp"
#include "vmc_common.hpp"

namespace vmc {
namespace {

// Inclusive scan over the wave in six DPP steps (row_shr 1, 2, 4, 8, then the last lane of
// the row before, then lane 31); op(v, 0) = v for the values scanned
template <typename Op>
__device__ __forceinline__ int wave_scan(int v, Op op) {
    v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true));
    v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true));
    v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true));
    v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true));
    v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));
    v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));
    return v;
}
// over the workgroup (NW waves at most); all: the last one's
template <int NW, typename Op>
__device__ __forceinline__ int block_scan(int v, int (&sh)[NW], Op op, int& all) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = blockDim.x >> 6;
    v = wave_scan(v, op);
    if (lane == 63) sh[w] = v;
    __syncthreads();
    int x[NW];
#pragma unroll
    for (int i = 0; i < NW; ++i) x[i] = sh[i];
    int run = 0, before = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        before = i < w ? op(run, x[i]) : before;
        run = i < nw ? op(run, x[i]) : run;
    }
    all = run;
    __syncthreads();
    return op(v, before);
}
__device__ __forceinline__ long long block_scan(long long v, long long* sh, long long& all) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = blockDim.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const long long o = __shfl_up(v, d, kWave);
        if (lane >= d) v += o;
    }
    if (lane == 63) sh[w] = v;
    __syncthreads();
    long long before = 0;
    all = 0;
    for (int i = 0; i < nw; ++i) {
        before += i < w ? sh[i] : 0;
        all += sh[i];
    }
    __syncthreads();
    return v + before;
}

template <typename T>
__device__ __forceinline__ T div_floor(T x, T y) {  // x >= 0, y > 0
    if constexpr (sizeof(T) == 4) return (T)((uint32_t)x / (uint32_t)y);
    else return ((x | y) >> 32) == 0 ? (T)((uint32_t)x / (uint32_t)y) : x / y;
}

// One set, from its length (group: shared tokens; sequence: states; row: tokens)
__device__ __forceinline__ SetDesc make_desc(const PlanParams& p, int i, int row0, int ntok, int len, int key0, int group,
                                             int shared) {
    SetDesc d = {};
    if (i < p.ns) {
        d.row0 = row0;
        d.ntok = ntok;
        const int n = max(len, 0);
        if (p.paged) {
            d.src = row0;
            // a group of one row has nothing to share: all its keys are the row's own
            d.khi = ntok > 1 ? min(n, p.max_keys) : 0;
        } else {
            const long long end = min((long long)key0 + n, (long long)p.num_keys);
            d.src = max(key0, 0);
            d.khi = (int)max(end - d.src, 0ll);
        }
    } else {
        d.row0 = d.src = i - p.ns;
        d.ntok = 1;
        d.khi = min(len, p.max_keys);
        d.klo = max(shared, 0);
        d.own = group + 2;  // 1: of no group
    }
    d.nb = (int)div_floor<long long>((long long)d.ntok * p.G + p.RB - 1, p.RB);
    d.tiles = d.ntok > 0 && d.khi > d.klo ? (int)(((long long)d.khi - (d.klo & ~15) + 63) / 64) : 0;
    return d;
}
// the group of a row that shares something with others, or -1: starts gs[0 .. ns]
__device__ __forceinline__ int group_of(const int* gs, int ns, int row) {
    int lo = 0, hi = ns + 1;  // starts that are <= row
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (gs[mid] <= row) lo = mid + 1;
        else hi = mid;
    }
    return lo >= 1 && lo <= ns && gs[lo] - gs[lo - 1] > 1 ? lo - 1 : -1;
}
// tiles before unit u of a set (and the first tile's place at or after u)
template <typename T>
__device__ __forceinline__ T tiles_before(const SetDesc& d, T cum, T cumt, T u, RangeRec& rec) {
    const T rem = u - cum, per = d.tiles + kItemCost, item = div_floor<T>(rem, per);
    rec.t = max((int)(rem - item * per) - kItemCost, 0);
    rec.g = (int)div_floor<T>(item, d.nb);
    rec.rb = (int)(item - (T)rec.g * d.nb);
    return cumt + item * d.tiles + rec.t;
}
// last set of n with cum <= u
template <typename T>
__device__ __forceinline__ int set_of(const T* cum, int n, T u) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cum[mid] <= u) lo = mid;
        else hi = mid;
    }
    return lo;
}
__device__ __forceinline__ RowRec make_row(const SetDesc& own, int64_t own_u, const SetDesc* desc, int64_t grp_u) {
    RowRec r = {};
    r.own_u = own_u;
    r.own_tiles = own.tiles;
    if (own.own > 1) {
        const SetDesc d = desc[own.own - 2];
        r.grp_u = grp_u;
        r.grp_tiles = d.tiles;
        r.grp_nb = d.nb;
        r.grp_row0 = d.row0;
        r.grp_ntok = d.ntok;
    }
    return r;
}

// ---- the short plan, a thread a set (MAXS sets at most, fewer than threads), units
// in 32 bits
template <int MAXS, int NW>
struct PlanLds {
    int sh[3][NW];
    int gs[MAXS + 1], len[MAXS], cum[MAXS], cumt[MAXS];
};
struct PlanSums {
    SetDesc d;           // set i's
    int cum;             // units before it
    int total, total_t;  // units, tiles of all
};
// Sets into desc and sums into lds, visible to all threads on return
template <int MAXS, int NW>
__device__ __forceinline__ PlanSums plan_sets(const PlanParams& p, PlanLds<MAXS, NW>& lds, SetDesc* desc, int i) {
    int len = 0, key0 = 0;
    if (i < p.ns) {
        len = p.set_lens[i];
        if (!p.paged) key0 = p.key_starts[i];
    } else if (i < p.nsets) {
        len = p.seq_lens[i - p.ns];
    }
    int all;
    const int start = p.ns > 0 && i <= p.ns ? min(max(p.starts[i], 0), p.rows) : 0;
    const int gs = block_scan(start, lds.sh[0], [](int a, int b) { return max(a, b); }, all);
    if (i <= p.ns) lds.gs[i] = gs;
    if (i < p.nsets) lds.len[i] = len;
    __syncthreads();
    PlanSums x = {};
    int units = 0, tiles = 0;
    if (i < p.nsets) {
        const int j = i < p.ns ? -1 : group_of(lds.gs, p.ns, i - p.ns);
        x.d = make_desc(p, i, i < p.ns ? lds.gs[i] : 0, i < p.ns ? lds.gs[i + 1] - lds.gs[i] : 0, len, key0, j,
                        j >= 0 ? lds.len[j] : 0);
        const int items = p.Hkv * x.d.nb;
        units = p.whole ? items : x.d.tiles ? items * (x.d.tiles + kItemCost) : 0;
        tiles = items * x.d.tiles;
        desc[i] = x.d;
    }
    x.cum = block_scan(units, lds.sh[1], [](int a, int b) { return a + b; }, x.total) - units;
    const int cumt = block_scan(tiles, lds.sh[2], [](int a, int b) { return a + b; }, x.total_t) - tiles;
    if (i < p.nsets) {
        lds.cum[i] = x.cum;
        lds.cumt[i] = cumt;
    }
    __syncthreads();
    return x;
}
// what the kernels behind the plan read of the sets
__device__ __forceinline__ void plan_out(const PlanParams& p, const PlanSums& x, const SetDesc* desc, const int* cum, int i) {
    if (i < p.nsets) {
        p.desc[i] = x.d;
        p.cum[i] = x.cum;
    }
    if (i == 0) p.cum[p.nsets] = x.total;
    if (p.paged && i >= p.ns && i < p.nsets)
        p.row[i - p.ns] = make_row(x.d, x.cum, desc, x.d.own > 1 ? cum[x.d.own - 2] : 0);
}
// the record of the range that begins at unit u, without its number of tiles; the
// tiles before it
template <int MAXS, int NW>
__device__ __forceinline__ int range_begin(const PlanLds<MAXS, NW>& lds, const SetDesc* desc, int nsets, int u, RangeRec& r) {
    r.set = set_of(lds.cum, nsets, u);
    r.d = desc[r.set];
    return tiles_before(r.d, lds.cum[r.set], lds.cumt[r.set], u, r);
}

}  // namespace
}  // namespace vmc
