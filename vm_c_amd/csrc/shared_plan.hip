// shared_plan.hip -- plan and merge kernels around the shared-keys kernel
// (shared_tile.hpp), and its launches.
//
// The plan is one workgroup's: lengths and starts live on the device, so a captured
// call follows them, and the kernels behind it find any unit of the axis by one or
// two rounds of 64 probes instead of scanning the batch each.
#include "shared_plan.hpp"

#include <algorithm>

#include "device_cus.hpp"
#include "vmc_common.hpp"

namespace vmc {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kUnitsMin = kItemCost + 1;  // fewest units of a range: one tile
constexpr int kPlanCached = 1024;  // sets that the plan keeps in LDS

// Inclusive scan over the workgroup of N values a thread by op; all: the last one's.
template <int N, typename T, typename Op>
__device__ __forceinline__ void block_incl_scan(T (&v)[N], T (*sh)[N], Op op, T (&all)[N]) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = blockDim.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1)
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const T o = __shfl_up(v[k], d, kWave);
            if (lane >= d) v[k] = op(v[k], o);
        }
    if (lane == 63)
#pragma unroll
        for (int k = 0; k < N; ++k) sh[w][k] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
        T run = sh[0][k], before = run;
        for (int i = 1; i < nw; ++i) {
            if (i == w) before = run;
            run = op(run, sh[i][k]);
        }
        if (w > 0) v[k] = op(before, v[k]);
        all[k] = run;
    }
    __syncthreads();
}

__device__ __forceinline__ int64_t div_small(int64_t x, int64_t y) {  // x, y >= 0; y > 0
    return ((x | y) >> 32) == 0 ? (int64_t)((uint32_t)x / (uint32_t)y) : x / y;
}

// tiles before unit u of a set (with the first tile's place at or after u in *rec)
__device__ __forceinline__ int64_t tiles_before(const SetDesc& d, int64_t cum, int64_t cumt, int64_t u, RangeRec* rec) {
    const int64_t rem = u - cum;
    const int per = d.tiles + kItemCost;
    const int64_t item = div_small(rem, per);
    const int x = max((int)(rem - item * per) - kItemCost, 0);
    if (rec) {
        rec->g = (int)div_small(item, d.nb);
        rec->rb = (int)(item - (int64_t)rec->g * d.nb);
        rec->t = x;
    }
    return cumt + item * d.tiles + x;
}

// CACHED: the sets fit the LDS copies, which later steps of the plan read instead of
// what it has just written
template <bool CACHED>
__global__ void __launch_bounds__(kPlanThreads) shared_plan_kernel(PlanParams p) {
    constexpr int NC = CACHED ? kPlanCached : 1;
    __shared__ int shi[kPlanThreads / 64][1];
    __shared__ long long shl[kPlanThreads / 64][2];
    __shared__ long long s_cum[NC + 1], s_cumt[NC + 1];
    __shared__ SetDesc s_desc[NC];
    __shared__ int s_gs[NC + 1];
    const int tid = threadIdx.x, nt = blockDim.x;
    // lengths of this thread's first set: on their way while the starts are scanned
    int len = 0, key0 = 0;
    auto lengths = [&](int i) {
        if (i < p.ns) {
            len = p.set_lens[i];
            if (!p.paged) key0 = p.key_starts[i];
        } else if (i < p.nsets) {
            len = p.seq_lens[i - p.ns];
        }
    };
    lengths(tid);
    int carry = 0;
    for (int i0 = 0; i0 <= p.ns; i0 += nt) {
        const int i = i0 + tid;
        int v[1] = {p.ns > 0 && i <= p.ns ? min(max(p.starts[i], 0), p.rows) : 0};
        int all[1];
        block_incl_scan<1>(v, shi, [](int a, int b) { return max(a, b); }, all);
        if (i <= p.ns) {
            p.gs[i] = max(carry, v[0]);
            if (CACHED) s_gs[i] = max(carry, v[0]);
        }
        carry = max(carry, all[0]);
    }
    __syncthreads();
    const int* gs = CACHED ? s_gs : p.gs;
    long long done[2] = {0, 0};  // units, tiles
    for (int i0 = 0; i0 < p.nsets; i0 += nt) {
        const int i = i0 + tid;
        if (i0) lengths(i);
        SetDesc d = {};
        long long amount[2] = {0, 0};
        if (i < p.nsets) {
            if (i < p.ns) {
                d.row0 = gs[i];
                d.ntok = gs[i + 1] - d.row0;
                const int n = max(len, 0);
                if (p.paged) {
                    d.src = d.row0;
                    // a group of one row has nothing to share: all its keys are the row's own
                    d.khi = d.ntok > 1 ? min(n, p.max_keys) : 0;
                } else {
                    const long long end = min((long long)key0 + n, (long long)p.num_keys);
                    d.src = max(key0, 0);
                    d.khi = (int)max(end - d.src, 0ll);
                }
            } else {
                d.row0 = d.src = i - p.ns;
                d.ntok = 1;
                d.khi = min(len, p.max_keys);
                int lo = 0, hi = p.ns + 1;  // starts that are <= row
                while (lo < hi) {
                    const int mid = (lo + hi) >> 1;
                    if (gs[mid] <= d.row0) lo = mid + 1;
                    else hi = mid;
                }
                const bool in = lo >= 1 && lo <= p.ns && gs[lo] - gs[lo - 1] > 1;
                if (in) d.klo = max(p.set_lens[lo - 1], 0);
                d.own = in ? lo + 1 : 1;  // 2 + its group
            }
            d.nb = (int)div_small((long long)d.ntok * p.G + p.RB - 1, p.RB);
            d.tiles = d.ntok > 0 && d.khi > d.klo ? (int)(((long long)d.khi - (d.klo & ~15) + 63) / 64) : 0;
            const long long items = (long long)p.Hkv * d.nb;
            amount[0] = p.whole ? items : d.tiles ? items * (d.tiles + kItemCost) : 0;
            amount[1] = items * d.tiles;
            p.desc[i] = d;
            if (CACHED) s_desc[i] = d;
        }
        long long incl[2] = {amount[0], amount[1]}, all[2];
        block_incl_scan<2>(incl, shl, [](long long a, long long b) { return a + b; }, all);
        if (i < p.nsets) {
            const long long u = done[0] + incl[0] - amount[0], v = done[1] + incl[1] - amount[1];
            p.cum[i] = u;
            if (CACHED) {
                s_cum[i] = u;
                s_cumt[i] = v;
            } else {
                p.cumt[i] = v;
            }
        }
        done[0] += all[0];
        done[1] += all[1];
    }
    if (tid == 0) p.cum[p.nsets] = done[0];
    if (p.whole) return;
    __syncthreads();
    const long long* cum = CACHED ? s_cum : reinterpret_cast<const long long*>(p.cum);
    const long long* cumt = CACHED ? s_cumt : reinterpret_cast<const long long*>(p.cumt);
    const SetDesc* desc = CACHED ? s_desc : p.desc;
    const long long total = done[0];
    const int n = plan_ranges(total, p.grid, p.umin);
    auto set_of = [&](long long u) {  // last set with cum <= u
        int lo = 0, hi = p.nsets;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (cum[mid] <= u) lo = mid;
            else hi = mid;
        }
        return lo;
    };
    for (int w = tid; w < p.grid; w += nt) {
        RangeRec r = {};
        if (w < n) {
            const long long u0 = div_small((long long)w * total, n), u1 = div_small((long long)(w + 1) * total, n);
            r.set = set_of(u0);
            r.d = desc[r.set];
            const int64_t t0 = tiles_before(r.d, cum[r.set], cumt[r.set], u0, &r);
            int64_t t1 = done[1];
            if (u1 < total) {
                const int s1 = set_of(u1);
                t1 = tiles_before(desc[s1], cum[s1], cumt[s1], u1, nullptr);
            }
            r.ntiles = (int)(t1 - t0);
        }
        p.range[w] = r;
    }
    if (!p.paged) return;
    for (int b = tid; b < p.rows; b += nt) {
        RowRec r = {};
        const SetDesc own = desc[p.ns + b];
        r.own_u = cum[p.ns + b];
        r.own_tiles = own.tiles;
        if (own.own > 1) {
            const int j = own.own - 2;
            const SetDesc d = desc[j];
            r.grp_u = cum[j];
            r.grp_tiles = d.tiles;
            r.grp_nb = d.nb;
            r.grp_row0 = d.row0;
            r.grp_ntok = d.ntok;
        }
        p.row[b] = r;
    }
}

// the pieces of a row: of ranges w0 .. w0 + cnt - 1, first partial row base (of range 0)
struct Pieces {
    int w0[2], cnt[2];
    int64_t base[2];
};

// sum over pieces first, first + step, .. of np: o, l against the running maximum m
template <int D, typename PieceAt>
__device__ __forceinline__ void merge_pieces(int first, int step, int np, int lane, PieceAt piece, float& m, float& l,
                                             float (&acc)[D / 64]) {
    constexpr int NPL = D / 64;
    typedef float vec __attribute__((ext_vector_type(NPL == 1 ? 2 : NPL)));
    m = -__builtin_inff();
    l = 0.0f;
#pragma unroll
    for (int e = 0; e < NPL; ++e) acc[e] = 0.0f;
    constexpr int U = 8;
    for (int i0 = first; i0 < np; i0 += U * step) {
        float x[U][NPL];
        float2 ml[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const float* s = piece(min(i0 + i * step, np - 1));
            ml[i] = *reinterpret_cast<const float2*>(s + D);
            if constexpr (NPL == 1) x[i][0] = s[lane];
            else {
                const vec y = *reinterpret_cast<const vec*>(s + NPL * lane);
#pragma unroll
                for (int e = 0; e < NPL; ++e) x[i][e] = y[e];
            }
        }
        float mx = m;
#pragma unroll
        for (int i = 0; i < U; ++i) mx = fmaxf(mx, i0 + i * step < np ? ml[i].x : -__builtin_inff());
        const float a = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - mx);
        m = mx;
        l = a == 0.0f ? 0.0f : l * a;
#pragma unroll
        for (int e = 0; e < NPL; ++e) acc[e] = a == 0.0f ? 0.0f : acc[e] * a;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            // (a piece of weight 0 adds nothing, not 0 * inf; a NaN reference stays one)
            const bool in = i0 + i * step < np && ml[i].x != -__builtin_inff();
            const float wt = in ? __builtin_amdgcn_exp2f(ml[i].x - mx) : 0.0f;
            l = wt == 0.0f ? l : __builtin_fmaf(wt, ml[i].y, l);
#pragma unroll
            for (int e = 0; e < NPL; ++e) acc[e] = wt == 0.0f ? acc[e] : __builtin_fmaf(wt, x[i][e], acc[e]);
        }
    }
}

// Paged calls: one workgroup per row and query head; its waves take every fourth piece
// of the group's common keys and of the row's own.
template <int D, bool BF>
__global__ void __launch_bounds__(256) shared_merge_paged_kernel(TileParams p, int RB) {
    constexpr int NPL = D / 64;
    __shared__ float so[4][D], sml[4][2];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = blockIdx.x / p.Hq, hq = blockIdx.x % p.Hq, g = hq / p.G;
    const int64_t total = p.cum[p.nsets];
    const RowRec rec = p.row[b];
    const int n = plan_ranges(total, p.grid, p.umin);
    Pieces pc = {};
    if (rec.grp_tiles) {
        const int r = (b - rec.grp_row0) * p.G + hq % p.G, rb = r / RB;
        const int64_t u = rec.grp_u + ((int64_t)g * rec.grp_nb + rb) * (rec.grp_tiles + kItemCost) + kItemCost;
        pc.w0[0] = plan_range_of(u, total, n);
        pc.cnt[0] = plan_range_of(u + rec.grp_tiles - 1, total, n) - pc.w0[0] + 1;
        pc.base[0] = plan_rows_paged(0, RB, p.Hq, p.G, p.total_rows, 0, rec.grp_row0, rec.grp_ntok, g, rb) + r % RB;
    }
    if (rec.own_tiles) {
        const int r = hq % p.G, rb = r / RB, nb = (p.G + RB - 1) / RB;
        const int64_t u = rec.own_u + ((int64_t)g * nb + rb) * (rec.own_tiles + kItemCost) + kItemCost;
        pc.w0[1] = plan_range_of(u, total, n);
        pc.cnt[1] = plan_range_of(u + rec.own_tiles - 1, total, n) - pc.w0[1] + 1;
        pc.base[1] = plan_rows_paged(0, RB, p.Hq, p.G, p.total_rows, 1, b, 1, g, rb) + r % RB;
    }
    auto piece = [&](int i) __attribute__((always_inline)) -> const float* {
        const int k = i >= pc.cnt[0] ? 1 : 0;
        const int at = (k ? pc.w0[1] - pc.cnt[0] : pc.w0[0]) + i;
        return p.part + ((int64_t)at * RB + (k ? pc.base[1] : pc.base[0])) * (D + 4);
    };
    float m, l, acc[NPL];
    merge_pieces<D>(w, 4, pc.cnt[0] + pc.cnt[1], lane, piece, m, l, acc);
#pragma unroll
    for (int e = 0; e < NPL; ++e) so[w][NPL * lane + e] = acc[e];
    if (lane == 0) {
        sml[w][0] = m;
        sml[w][1] = l;
    }
    __syncthreads();
    if (threadIdx.x >= D) return;
    float mx = sml[0][0];
#pragma unroll
    for (int i = 1; i < 4; ++i) mx = fmaxf(mx, sml[i][0]);
    float o = 0.0f, ls = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float wt = sml[i][0] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(sml[i][0] - mx);
        o = wt == 0.0f ? o : __builtin_fmaf(wt, so[i][threadIdx.x], o);
        ls = wt == 0.0f ? ls : __builtin_fmaf(wt, sml[i][1], ls);
    }
    p.out[(int64_t)blockIdx.x * D + threadIdx.x] = f32_to_half<BF>(ls == 0.0f ? 0.0f : o / ls);
}

// Contiguous calls: workgroup (x, y) has the item that range x begins and does not
// finish, if there is one (whole items are written already), and 16 of its
// rows; and sets without keys, whose rows are zero.
template <int D, bool BF>
__global__ void __launch_bounds__(256) shared_merge_local_kernel(TileParams p, int RB) {
    constexpr int NPL = D / 64;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int w = blockIdx.x;
    for (int s = w; s < p.ns; s += p.grid) {
        const SetDesc d = p.desc[s];
        if (d.tiles) continue;
        const int64_t n = (int64_t)d.ntok * p.Hq * D / 8;
        for (int64_t i = (int64_t)blockIdx.y * 256 + threadIdx.x; i < n; i += 256 * (int64_t)gridDim.y)
            *reinterpret_cast<u32x4*>(p.out + (int64_t)d.row0 * p.Hq * D + 8 * i) = u32x4{0u, 0u, 0u, 0u};
    }
    if (w + 1 >= p.grid) return;
    const RangeRec rec = p.range[w + 1], me = p.range[w];
    // the next range begins inside an item, which began here: not before this range
    if (rec.t == 0 || (me.set == rec.set && me.g == rec.g && me.rb == rec.rb && me.t > 0)) return;
    const int nrow = min(RB, rec.d.ntok * p.G - RB * rec.rb), r0 = 16 * blockIdx.y + 4 * wv;
    if (r0 >= nrow) return;
    const int64_t total = p.cum[p.nsets];
    const int n = plan_ranges(total, p.grid, p.umin);
    const int64_t last = p.cum[rec.set] + ((int64_t)rec.g * rec.d.nb + rec.rb + 1) * (rec.d.tiles + kItemCost) - 1;
    const int cnt = plan_range_of(last, total, n) - w + 1;
    for (int r = r0; r < min(r0 + 4, nrow); ++r) {
        auto piece = [&](int i) __attribute__((always_inline)) -> const float* {
            return p.part + (plan_rows_local(w + i, RB, i > 0) + r) * (D + 4);
        };
        float m, l, acc[NPL];
        merge_pieces<D>(0, 1, cnt, lane, piece, m, l, acc);
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        const int x = RB * rec.rb + r;
        uint16_t* op = p.out + ((rec.d.row0 + x / p.G) * (int64_t)p.Hq + rec.g * p.G + x % p.G) * D + NPL * lane;
#pragma unroll
        for (int e = 0; e < NPL; ++e) op[e] = f32_to_half<BF>(acc[e] * inv);
    }
}

template <int D, bool BF>
void launch_merge_d(const TileParams& p, int RB, hipStream_t s) {
    if (p.paged) {
        const int64_t rows = (int64_t)p.total_rows * p.Hq;
        hipLaunchKernelGGL((shared_merge_paged_kernel<D, BF>), dim3((unsigned)rows), dim3(256), 0, s, p, RB);
        return;
    }
    hipLaunchKernelGGL((shared_merge_local_kernel<D, BF>), dim3((unsigned)p.grid, (unsigned)RB / 16), dim3(256), 0, s, p,
                       RB);
}

int launch_merge(const TileParams& p, int D, bool bf, int RB, hipStream_t s) {
    switch (D) {
        case 64: bf ? launch_merge_d<64, true>(p, RB, s) : launch_merge_d<64, false>(p, RB, s); break;
        case 128: bf ? launch_merge_d<128, true>(p, RB, s) : launch_merge_d<128, false>(p, RB, s); break;
        default: bf ? launch_merge_d<256, true>(p, RB, s) : launch_merge_d<256, false>(p, RB, s); break;
    }
    VMC_LAUNCH_CHECK();
    return VMC_OK;
}

// How a call runs, from its sizes alone (lengths are on the device).
struct Shape {
    int whole, grid;  // one item a workgroup; ranges (whole: workgroups)
    bool conv;        // bf16 V is converted to fp16
    size_t cum, cumt, desc, range, row, gs, part, bytes;  // workspace offsets, size
};

Shape shape_of(bool paged, int rows, int nsets, int Hq, int Hkv, int D) {
    Shape sh = {};
    const int64_t G = Hq / Hkv, sets = std::max(nsets, 1);
    // workgroups that fit a CU: 64 KB of tiles each (head_dim 256: 128 KB)
    sh.grid = num_cus() * (D == 256 ? 1 : 2);
    // Whole items where sets of many rows give several times the workgroups
    const int64_t items = (int64_t)Hkv * (rows * G / kTileRows + std::min<int64_t>(rows, sets));
    if (!paged && rows * G >= kTileRows * sets && items >= 4 * (int64_t)sh.grid && items < (1 << 30)) {
        sh.whole = 1;
        sh.grid = (int)((items + 7) & ~7);
    }
    sh.conv = rows * G >= 64 * sets;
    const int64_t total = paged ? (int64_t)nsets + rows : nsets;
    const int64_t prow = sh.whole ? 0 : paged ? (int64_t)sh.grid * kTileRows + 2 * (int64_t)rows * Hq : 2 * (int64_t)sh.grid * kTileRows;
    auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    sh.cum = 0;
    sh.cumt = up((size_t)(total + 1) * sizeof(int64_t));
    sh.desc = 2 * sh.cumt;
    sh.range = sh.desc + up((size_t)total * sizeof(SetDesc));
    sh.row = sh.range + (sh.whole ? 0 : up((size_t)sh.grid * sizeof(RangeRec)));
    sh.gs = sh.row + (paged ? up((size_t)rows * sizeof(RowRec)) : 0);
    sh.part = sh.gs + up((size_t)(nsets + 1) * sizeof(int32_t));
    sh.bytes = sh.part + (size_t)prow * (D + 4) * sizeof(float);
    return sh;
}

}  // namespace

size_t shared_tiles_workspace(bool paged, int rows, int nsets, int Hq, int Hkv, int D) {
    return shape_of(paged, rows, nsets, Hq, Hkv, D).bytes;
}

bool shared_tiles_take(const SharedArgs& a) {
    if (((uintptr_t)a.q & 15) != 0 || ((uintptr_t)a.out & 15) != 0 || a.q_ts % 8 != 0 || a.q_hs % 8 != 0) return false;
    if (a.src == GEN_LOCAL)
        return (((uintptr_t)a.k | (uintptr_t)a.v) & 15) == 0 && a.k_ts % 8 == 0 && a.k_hs % 8 == 0 && a.v_ts % 8 == 0 &&
               a.v_hs % 8 == 0 && a.k_ts < (1 << 23) && a.v_ts < (1 << 23);
    if (a.bs % 16 != 0 || (a.hnd ? 1 : a.Hkv) * a.entry * 16 > 0x7fffffff) return false;
    if (a.src == GEN_F16 || a.src == GEN_BF16)
        return (a.src == GEN_BF16) == (a.q_bf16 != 0) && (((uintptr_t)a.kp | (uintptr_t)a.vp) & 15) == 0;
    return (((uintptr_t)a.kp | (uintptr_t)a.vp) & 3) == 0;
}

int shared_tiles(const SharedArgs& a, void* ws, hipStream_t s) {
    const bool paged = a.src != GEN_LOCAL;
    const Shape sh = shape_of(paged, a.rows, a.nsets, a.Hq, a.Hkv, a.D);
    uint8_t* w = reinterpret_cast<uint8_t*>(ws);
    PlanParams pl = {};
    pl.starts = a.starts;
    pl.set_lens = a.set_lens;
    pl.seq_lens = a.seq_lens;
    pl.key_starts = a.key_starts;
    pl.ns = a.nsets;
    pl.rows = a.rows;
    pl.nsets = paged ? a.nsets + a.rows : a.nsets;
    pl.max_keys = (int)(a.max_blocks * a.bs);
    pl.num_keys = a.num_keys;
    pl.Hkv = a.Hkv;
    pl.G = a.Hq / a.Hkv;
    pl.RB = kTileRows;
    pl.paged = paged;
    pl.whole = sh.whole;
    pl.cum = reinterpret_cast<int64_t*>(w + sh.cum);
    pl.cumt = reinterpret_cast<int64_t*>(w + sh.cumt);
    pl.desc = reinterpret_cast<SetDesc*>(w + sh.desc);
    pl.range = reinterpret_cast<RangeRec*>(w + sh.range);
    pl.row = reinterpret_cast<RowRec*>(w + sh.row);
    pl.grid = sh.grid;
    pl.umin = kUnitsMin;
    pl.gs = reinterpret_cast<int32_t*>(w + sh.gs);
    const int threads = pl.nsets > 512 || sh.grid > 512 ? kPlanThreads : 512;
    if (pl.nsets <= kPlanCached) hipLaunchKernelGGL(shared_plan_kernel<true>, dim3(1), dim3(threads), 0, s, pl);
    else hipLaunchKernelGGL(shared_plan_kernel<false>, dim3(1), dim3(threads), 0, s, pl);
    VMC_LAUNCH_CHECK();

    TileParams p = {};
    p.out = a.out;
    p.q = a.q;
    p.q_ts = a.q_ts;
    p.q_hs = a.q_hs;
    p.Hq = a.Hq;
    p.Hkv = a.Hkv;
    p.G = pl.G;
    p.scale = a.scale;
    p.cum = pl.cum;
    p.desc = pl.desc;
    p.range = pl.range;
    p.row = pl.row;
    p.gs = pl.gs;
    p.ns = a.nsets;
    p.nsets = pl.nsets;
    p.paged = paged;
    p.whole = sh.whole;
    p.total_rows = a.rows;
    p.grid = sh.grid;
    p.umin = kUnitsMin;
    p.part = reinterpret_cast<float*>(w + sh.part);
    if (paged) {
        p.kp = a.kp;
        p.vp = a.vp;
        p.k_row = p.v_row = a.hnd ? a.entry : a.Hkv * a.entry;
        p.k_head = p.v_head = a.hnd ? a.bs * a.entry : a.entry;
        p.page_bytes = a.bs * a.Hkv * a.entry;
        p.max_blocks = a.max_blocks;
        p.bs = (int)a.bs;
        p.bt = a.bt;
        p.seq_lens = a.seq_lens;
    } else {
        p.kp = reinterpret_cast<const uint8_t*>(a.k);
        p.vp = reinterpret_cast<const uint8_t*>(a.v);
        p.k_row = 2 * a.k_ts;
        p.k_head = 2 * a.k_hs;
        p.v_row = 2 * a.v_ts;
        p.v_head = 2 * a.v_hs;
    }
    const int src = !paged ? 0 : a.src == GEN_Q8 ? 2 : a.src == GEN_Q4 ? 3 : 1;
    const bool bf = a.q_bf16 != 0;
    const int rc = a.D == 64    ? shared_tile_d64(p, src, bf, sh.conv, sh.grid, s)
                   : a.D == 128 ? shared_tile_d128(p, src, bf, sh.conv, sh.grid, s)
                                : shared_tile_d256(p, src, bf, sh.conv, sh.grid, s);
    if (rc != VMC_OK || sh.whole) return rc;
    return launch_merge(p, a.D, bf, pl.RB, s);
}

}  // namespace vmc
