// shared_plan.hip -- plan and merge kernels around the shared-keys kernel
// (shared_tile.hpp), and its launches.
//
// The plan is one workgroup's: lengths and starts live on the device, so a captured
// call follows them, and the kernels behind it find any unit of the axis by one or
// two rounds of 64 probes instead of scanning the batch each.
#include "shared_plan_dev.hpp"

#include <algorithm>

#include "device_cus.hpp"
#include "vmc_common.hpp"

namespace vmc {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanCached = 1024;         // sets, and ranges, that the short plan holds in LDS

// The plan of a call of at most kPlanCached sets and ranges whose units fit 32 bits, a
// thread a set: every step from registers and LDS.  What bounds it: its chain of
// dependent steps.
__global__ void __launch_bounds__(kPlanThreads) shared_plan_kernel(PlanParams p) {
    __shared__ PlanLds<kPlanCached, kPlanThreads / 64> lds;
    __shared__ int s_first[kPlanCached + 1];  // tiles before each range
    __shared__ SetDesc s_desc[kPlanCached];
    const int i = threadIdx.x;
    const PlanSums x = plan_sets(p, lds, s_desc, i);
    plan_out(p, x, s_desc, lds.cum, i);
    if (p.whole) return;
    const int n = plan_ranges(x.total, p.grid, p.cus);
    RangeRec r = {};
    if (i < n) {
        r.ntiles = range_begin(lds, s_desc, p.nsets, (int)div_floor<long long>((long long)i * x.total, n), r);
        s_first[i] = r.ntiles;
    }
    if (i == 0) s_first[n] = x.total_t;
    __syncthreads();
    if (i < n) r.ntiles = s_first[i + 1] - r.ntiles;
    if (i < p.grid) p.range[i] = r;
}

// The plan of any other call, through memory
__global__ void __launch_bounds__(kPlanThreads) shared_plan_long_kernel(PlanParams p) {
    __shared__ int shi[16];
    __shared__ long long shl[16];
    const int tid = threadIdx.x, nt = blockDim.x;
    int carry = 0;
    for (int i0 = 0; i0 <= p.ns; i0 += nt) {
        const int i = i0 + tid;
        int all;
        const int v = block_scan(p.ns > 0 && i <= p.ns ? min(max(p.starts[i], 0), p.rows) : 0, shi,
                                 [](int a, int b) { return max(a, b); }, all);
        if (i <= p.ns) p.gs[i] = max(carry, v);
        carry = max(carry, all);
    }
    __syncthreads();
    long long total = 0, total_t = 0;
    for (int i0 = 0; i0 < p.nsets; i0 += nt) {
        const int i = i0 + tid;
        long long units = 0, tiles = 0;
        if (i < p.nsets) {
            SetDesc d;
            if (i < p.ns) {
                d = make_desc(p, i, p.gs[i], p.gs[i + 1] - p.gs[i], p.set_lens[i], p.paged ? 0 : p.key_starts[i], -1, 0);
            } else {
                const int j = group_of(p.gs, p.ns, i - p.ns);
                d = make_desc(p, i, 0, 0, p.seq_lens[i - p.ns], 0, j, j >= 0 ? p.set_lens[j] : 0);
            }
            const long long items = (long long)p.Hkv * d.nb;
            units = p.whole ? items : d.tiles ? items * (d.tiles + kItemCost) : 0;
            tiles = items * d.tiles;
            p.desc[i] = d;
        }
        long long all, all_t;
        const long long cum = block_scan(units, shl, all) - units, cumt = block_scan(tiles, shl, all_t) - tiles;
        if (i < p.nsets) {
            p.cum[i] = total + cum;
            p.cumt[i] = total_t + cumt;
        }
        total += all;
        total_t += all_t;
    }
    if (tid == 0) p.cum[p.nsets] = total;
    if (p.whole) return;
    __syncthreads();
    const int n = plan_ranges(total, p.grid, p.cus);
    for (int w = tid; w < p.grid; w += nt) {
        RangeRec r = {}, e = {};
        if (w < n) {
            const int64_t u0 = div_floor<int64_t>((int64_t)w * total, n), u1 = div_floor<int64_t>((int64_t)(w + 1) * total, n);
            r.set = set_of<int64_t>(p.cum, p.nsets, u0);
            r.d = p.desc[r.set];
            const int64_t t0 = tiles_before<int64_t>(r.d, p.cum[r.set], p.cumt[r.set], u0, r);
            int64_t t1 = total_t;
            if (u1 < total) {
                const int s = set_of<int64_t>(p.cum, p.nsets, u1);
                t1 = tiles_before<int64_t>(p.desc[s], p.cum[s], p.cumt[s], u1, e);
            }
            r.ntiles = (int)(t1 - t0);
        }
        p.range[w] = r;
    }
    if (!p.paged) return;
    for (int b = tid; b < p.rows; b += nt) {
        const SetDesc own = p.desc[p.ns + b];
        p.row[b] = make_row(own, p.cum[p.ns + b], p.desc, own.own > 1 ? p.cum[own.own - 2] : 0);
    }
}

// ---- merge.  A row of D values is D / 4 lanes of 16 bytes, so that a workgroup has
// 1024 / D rows of lanes.

// pieces first, first + step, .. of np into o, l against their largest reference m
template <typename PieceAt>
__device__ __forceinline__ void merge_pieces(int first, int step, int np, int D, int lane, PieceAt piece, float& m,
                                             float& l, f32x4& o) {
    m = -__builtin_inff();
    l = 0.0f;
    o = f32x4{0.f, 0.f, 0.f, 0.f};
    constexpr int U = 4;
    for (int i0 = first; i0 < np; i0 += U * step) {
        f32x4 x[U];
        float2 ml[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const float* s = piece(min(i0 + i * step, np - 1));
            ml[i] = *reinterpret_cast<const float2*>(s + D);
            x[i] = *reinterpret_cast<const f32x4*>(s + 4 * lane);
        }
        float mx = m;
#pragma unroll
        for (int i = 0; i < U; ++i) mx = fmaxf(mx, i0 + i * step < np ? ml[i].x : -__builtin_inff());
        const float a = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - mx);
        m = mx;
        l = a == 0.0f ? 0.0f : l * a;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = a == 0.0f ? 0.0f : o[e] * a;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            // (a piece of weight 0 adds nothing, not 0 * inf; a NaN reference stays one)
            const bool in = i0 + i * step < np && ml[i].x != -__builtin_inff();
            const float wt = in ? __builtin_amdgcn_exp2f(ml[i].x - mx) : 0.0f;
            l = wt == 0.0f ? l : __builtin_fmaf(wt, ml[i].y, l);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = wt == 0.0f ? o[e] : __builtin_fmaf(wt, x[i][e], o[e]);
        }
    }
}

template <bool BF>
__device__ __forceinline__ u32x2 pack_row4(f32x4 o, float l) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    return u32x2{(uint32_t)f32_to_half<BF>(o[0] * inv) | ((uint32_t)f32_to_half<BF>(o[1] * inv) << 16),
                 (uint32_t)f32_to_half<BF>(o[2] * inv) | ((uint32_t)f32_to_half<BF>(o[3] * inv) << 16)};
}

// Paged calls: one workgroup per row and query head, the pieces of the group's common
// keys and of the row's own spread over its rows of lanes.
template <int D, bool BF>
__global__ void __launch_bounds__(256) shared_merge_paged_kernel(TileParams p, int RB) {
    constexpr int LR = D / 4, NG = 256 / LR;
    __shared__ __attribute__((aligned(16))) float so[NG][D];
    __shared__ float2 sml[NG];
    const int lane = threadIdx.x % LR, grp = threadIdx.x / LR;
    const int b = blockIdx.x / p.Hq, hq = blockIdx.x % p.Hq, g = hq / p.G;
    const int64_t total = p.cum[p.nsets];
    const RowRec rec = p.row[b];
    const int n = plan_ranges(total, p.grid, p.cus);
    int w0[2] = {0, 0}, cnt[2] = {0, 0};  // first range and pieces: common keys, own keys
    int64_t base[2] = {0, 0};             // partial row of range 0
    if (rec.grp_tiles) {
        const int r = (b - rec.grp_row0) * p.G + hq % p.G, rb = r / RB;
        const int64_t u = rec.grp_u + ((int64_t)g * rec.grp_nb + rb) * (rec.grp_tiles + kItemCost) + kItemCost;
        w0[0] = plan_range_of(u, total, n);
        cnt[0] = plan_range_of(u + rec.grp_tiles - 1, total, n) - w0[0] + 1;
        base[0] = plan_rows_paged(0, RB, p.Hq, p.G, p.total_rows, 0, rec.grp_row0, rec.grp_ntok, g, rb) + r % RB;
    }
    if (rec.own_tiles) {
        const int r = hq % p.G, rb = r / RB, nb = (p.G + RB - 1) / RB;
        const int64_t u = rec.own_u + ((int64_t)g * nb + rb) * (rec.own_tiles + kItemCost) + kItemCost;
        w0[1] = plan_range_of(u, total, n);
        cnt[1] = plan_range_of(u + rec.own_tiles - 1, total, n) - w0[1] + 1;
        base[1] = plan_rows_paged(0, RB, p.Hq, p.G, p.total_rows, 1, b, 1, g, rb) + r % RB;
    }
    auto piece = [&](int i) __attribute__((always_inline)) -> const float* {
        const int k = i >= cnt[0] ? 1 : 0;
        const int at = (k ? w0[1] - cnt[0] : w0[0]) + i;
        return p.part + ((int64_t)at * RB + (k ? base[1] : base[0])) * (D + 4);
    };
    float m, l;
    f32x4 o;
    merge_pieces(grp, NG, cnt[0] + cnt[1], D, lane, piece, m, l, o);
    *reinterpret_cast<f32x4*>(&so[grp][4 * lane]) = o;
    if (lane == 0) sml[grp] = make_float2(m, l);
    __syncthreads();
    if (threadIdx.x >= LR) return;
    float2 x[NG];
    float mx = -__builtin_inff(), ls = 0.0f;
#pragma unroll
    for (int i = 0; i < NG; ++i) {
        x[i] = sml[i];
        mx = fmaxf(mx, x[i].x);
    }
    o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NG; ++i) {
        const float wt = x[i].x == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(x[i].x - mx);
        const f32x4 y = *reinterpret_cast<const f32x4*>(&so[i][4 * lane]);
        ls = wt == 0.0f ? ls : __builtin_fmaf(wt, x[i].y, ls);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = wt == 0.0f ? o[e] : __builtin_fmaf(wt, y[e], o[e]);
    }
    *reinterpret_cast<u32x2*>(p.out + (int64_t)blockIdx.x * D + 4 * lane) = pack_row4<BF>(o, ls);
}

// Contiguous calls: workgroups (x, y) have the item that range x begins and does not
// finish, if there is one (whole items are written already), 1024 / D of its
// rows at a time; and sets without keys, whose rows are zero.
template <int D, bool BF>
__global__ void __launch_bounds__(256) shared_merge_local_kernel(TileParams p, int RB) {
    constexpr int LR = D / 4, NG = 256 / LR;
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
    const int lane = threadIdx.x % LR, nrow = min(RB, rec.d.ntok * p.G - RB * rec.rb);
    const int64_t total = p.cum[p.nsets];
    const int n = plan_ranges(total, p.grid, p.cus);
    const int64_t last = p.cum[rec.set] + ((int64_t)rec.g * rec.d.nb + rec.rb + 1) * (rec.d.tiles + kItemCost) - 1;
    const int cnt = plan_range_of(last, total, n) - w + 1;
    for (int r = NG * blockIdx.y + threadIdx.x / LR; r < nrow; r += NG * gridDim.y) {
        auto piece = [&](int i) __attribute__((always_inline)) -> const float* {
            return p.part + (plan_rows_local(w + i, RB, i > 0) + r) * (D + 4);
        };
        float m, l;
        f32x4 o;
        merge_pieces(0, 1, cnt, D, lane, piece, m, l, o);
        const int x = RB * rec.rb + r;
        *reinterpret_cast<u32x2*>(p.out + ((rec.d.row0 + x / p.G) * (int64_t)p.Hq + rec.g * p.G + x % p.G) * D +
                                  4 * lane) = pack_row4<BF>(o, l);
    }
}

template <int D, bool BF>
void launch_merge_d(const TileParams& p, int RB, hipStream_t s) {
    if (p.paged) {
        const int64_t rows = (int64_t)p.total_rows * p.Hq;
        hipLaunchKernelGGL((shared_merge_paged_kernel<D, BF>), dim3((unsigned)rows), dim3(256), 0, s, p, RB);
        return;
    }
    // workgroups for twice the rows of an even batch, 32 at least: as many as full items need
    // took 5.0 instead of 4.2 us where 8 sequences have one row a head, 8.1 instead of 5.5
    // where 16 have 8 of head_dim 256
    const int64_t rows = std::min<int64_t>(RB, std::max<int64_t>(32, 2 * (int64_t)p.total_rows * p.G / std::max(p.ns, 1)));
    hipLaunchKernelGGL((shared_merge_local_kernel<D, BF>), dim3((unsigned)p.grid, (unsigned)((rows * D + 1023) / 1024)), dim3(256),
                       0, s, p, RB);
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
    size_t cum, cumt, desc, range, row, gs, part, bytes;  // workspace offsets, size
};

Shape shape_of(bool paged, int rows, int nsets, int Hq, int Hkv, int D) {
    Shape sh = {};
    const int64_t G = Hq / Hkv, sets = std::max(nsets, 1);
    sh.grid = num_cus() * tile_per_cu(D);
    // Whole items where sets of many rows give several times the workgroups: 8 x 1024 rows over
    // 2048 states take 459 us with the plan, 503 as ranges with the merge; with fewer items
    // the last workgroups' share shows
    const int64_t items = (int64_t)Hkv * (rows * G / kTileRows + std::min<int64_t>(rows, sets));
    if (!paged && rows * G >= kTileRows * sets && items >= 4 * (int64_t)sh.grid && items < (1 << 24)) {
        sh.whole = 1;
        sh.grid = (int)((items + 7) & ~7);
    }
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
    pl.RB = a.src == GEN_Q8 || a.src == GEN_Q4 ? kTileRows / 2 : kTileRows;
    pl.paged = paged;
    pl.whole = sh.whole;
    pl.cum = reinterpret_cast<int64_t*>(w + sh.cum);
    pl.cumt = reinterpret_cast<int64_t*>(w + sh.cumt);
    pl.desc = reinterpret_cast<SetDesc*>(w + sh.desc);
    pl.range = reinterpret_cast<RangeRec*>(w + sh.range);
    pl.row = reinterpret_cast<RowRec*>(w + sh.row);
    pl.grid = sh.grid;
    pl.cus = num_cus();
    pl.gs = reinterpret_cast<int32_t*>(w + sh.gs);
    // units fit 32 bits where even the longest sets that fit the call do
    const int64_t tiles = paged ? pl.max_keys / 64 + 2 : a.num_keys / 64 + 2;
    const int64_t items = (int64_t)a.Hkv * (((int64_t)a.rows * pl.G / pl.RB + a.nsets) + (paged ? (int64_t)a.rows * ((pl.G - 1) / pl.RB + 1) : 0));
    const bool short_units = items < 0x7fffffff / (tiles + kItemCost);
    const int need = std::max({pl.nsets, a.nsets + 1, sh.whole ? 1 : sh.grid + 1});
    const bool fused = short_units && !sh.whole && std::max(pl.nsets, a.nsets + 1) <= kPlanFused;
    if (!fused) {
        if (short_units && need <= kPlanCached)
            hipLaunchKernelGGL(shared_plan_kernel, dim3(1), dim3((unsigned)(need + 63) / 64 * 64), 0, s, pl);
        else
            hipLaunchKernelGGL(shared_plan_long_kernel, dim3(1), dim3(kPlanThreads), 0, s, pl);
        VMC_LAUNCH_CHECK();
    }

    TileParams p = {};
    p.plan = pl;
    p.fused = fused;
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
    p.ns = a.nsets;
    p.nsets = pl.nsets;
    p.paged = paged;
    p.whole = sh.whole;
    p.total_rows = a.rows;
    p.grid = sh.grid;
    p.cus = pl.cus;
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
    const int rc = a.D == 64    ? shared_tile_d64(p, src, bf, sh.grid, s)
                   : a.D == 128 ? shared_tile_d128(p, src, bf, sh.grid, s)
                                : shared_tile_d256(p, src, bf, sh.grid, s);
    if (rc != VMC_OK || sh.whole) return rc;
    return launch_merge(p, a.D, bf, pl.RB, s);
}

}  // namespace vmc
