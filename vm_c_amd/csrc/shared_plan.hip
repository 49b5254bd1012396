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

template <typename T, typename Op>
__device__ __forceinline__ T block_incl_scan(T v, T* sh, Op op, T* total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const T o = __shfl_up(v, d, kWave);
        if (lane >= d) v = op(v, o);
    }
    if (lane == 63) sh[w] = v;
    __syncthreads();
    T all = sh[0];
    T before = sh[0];
#pragma unroll
    for (int i = 1; i < kPlanThreads / 64; ++i) {
        if (i < w) before = op(before, sh[i]);
        all = op(all, sh[i]);
    }
    if (w > 0) v = op(before, v);
    *total = all;
    __syncthreads();
    return v;
}

__global__ void __launch_bounds__(kPlanThreads) shared_plan_kernel(PlanParams p) {
    __shared__ int shi[kPlanThreads / 64];
    __shared__ long long shl[kPlanThreads / 64];
    const int tid = threadIdx.x;
    int carry = 0;
    for (int i0 = 0; i0 <= p.ns; i0 += kPlanThreads) {
        const int i = i0 + tid;
        int v = p.ns > 0 && i <= p.ns ? min(max(p.starts[i], 0), p.rows) : 0;
        int all;
        v = block_incl_scan(v, shi, [](int a, int b) { return max(a, b); }, &all);
        if (i <= p.ns) p.gs[i] = max(carry, v);
        carry = max(carry, all);
    }
    __syncthreads();
    long long done = 0;
    for (int i0 = 0; i0 < p.nsets; i0 += kPlanThreads) {
        const int i = i0 + tid;
        SetDesc d = {};
        long long amount = 0;
        if (i < p.nsets) {
            if (i < p.ns) {
                d.row0 = p.gs[i];
                d.ntok = p.gs[i + 1] - d.row0;
                const int n = max(p.set_lens[i], 0);
                if (p.paged) {
                    d.src = d.row0;
                    // a group of one row has nothing to share: all its keys are the row's own
                    d.khi = d.ntok > 1 ? min(n, p.max_keys) : 0;
                } else {
                    const long long end = min((long long)p.key_starts[i] + n, (long long)p.num_keys);
                    d.src = max(p.key_starts[i], 0);
                    d.khi = (int)max(end - d.src, 0ll);
                }
            } else {
                d.row0 = d.src = i - p.ns;
                d.ntok = d.own = 1;
                d.khi = min(p.seq_lens[d.row0], p.max_keys);
                int lo = 0, hi = p.ns + 1;  // starts that are <= row
                while (lo < hi) {
                    const int mid = (lo + hi) >> 1;
                    if (p.gs[mid] <= d.row0) lo = mid + 1;
                    else hi = mid;
                }
                if (lo >= 1 && lo <= p.ns && p.gs[lo] - p.gs[lo - 1] > 1) d.klo = max(p.set_lens[lo - 1], 0);
            }
            d.nb = (int)(((long long)d.ntok * p.G + p.RB - 1) / p.RB);
            d.tiles = d.khi > d.klo ? (int)(((long long)d.khi - (d.klo & ~15) + 63) / 64) : 0;
            amount = (long long)p.Hkv * d.nb * (p.whole ? 1 : d.tiles);
            p.desc[i] = d;
        }
        long long all;
        const long long incl = block_incl_scan(amount, shl, [](long long a, long long b) { return a + b; }, &all);
        if (i < p.nsets) p.cum[i] = done + incl - amount;
        done += all;
    }
    if (tid == 0) p.cum[p.nsets] = done;
}

// One wave per query head of a row: the pieces' rows, weighted by their maxima.
// Paged: pieces of the group's common keys and of the row's own; contiguous: of
// an item that ranges cut (whole ones are written already).
template <int D, bool BF>
__global__ void __launch_bounds__(256) shared_merge_kernel(TileParams p, int RB, int per_wave) {
    constexpr int NPL = D / 64;
    typedef float vec __attribute__((ext_vector_type(NPL == 1 ? 2 : NPL)));
    const int lane = threadIdx.x & 63;
    const int64_t total = p.cum[p.nsets];
    const int n = plan_ranges(total, p.grid, p.umin);
    const int64_t first = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * per_wave;
    for (int64_t row = first; row < min(first + per_wave, (int64_t)p.total_rows * p.Hq); ++row) {
        const int b = __builtin_amdgcn_readfirstlane((int)(row / p.Hq)), hq = __builtin_amdgcn_readfirstlane((int)(row % p.Hq));
        const int g = hq / p.G;
        int w0[2] = {0, 0}, cnt[2] = {0, 0};  // first range and pieces: common keys, own keys
        int64_t base[2] = {0, 0};             // partial row of range 0
        auto set_pieces = [&](int k, int s) __attribute__((always_inline)) {
            const SetDesc d = p.desc[s];
            if (d.tiles == 0) return;
            const int r = (b - d.row0) * p.G + hq % p.G, rb = r / RB;
            const int64_t u = p.cum[s] + ((int64_t)g * d.nb + rb) * d.tiles;
            w0[k] = plan_range_of(u, total, n);
            cnt[k] = plan_range_of(u + d.tiles - 1, total, n) - w0[k] + 1;
            base[k] = (p.paged ? plan_rows_paged(0, RB, p.Hq, p.G, p.total_rows, d, g, rb) : 0) + r % RB;
        };
        const int j = p.ns > 0 ? plan_find(p.gs, p.ns + 1, b, lane) : -1;
        const bool in_set = p.ns > 0 && p.gs[0] <= b && j < p.ns;
        if (in_set) set_pieces(0, j);
        if (p.paged) set_pieces(1, p.ns + b);
        else if (!in_set || cnt[0] == 1) continue;  // padding, or written
        const int np = cnt[0] + cnt[1];
        auto piece = [&](int i) __attribute__((always_inline)) -> const float* {
            const int k = i >= cnt[0] ? 1 : 0, w = w0[k] + i - (k ? cnt[0] : 0);
            const int64_t at = p.paged ? (int64_t)w * RB + base[k] : plan_rows_local(w, RB, i > 0) + base[0];
            return p.part + at * (D + 4);
        };
        float mx = -__builtin_inff();
        for (int i = lane; i < np; i += 64) mx = fmaxf(mx, piece(i)[D]);
#pragma unroll
        for (int m = 32; m >= 1; m >>= 1) mx = fmaxf(mx, shfl_xor(mx, m));
        float acc[NPL], l = 0.0f;
#pragma unroll
        for (int e = 0; e < NPL; ++e) acc[e] = 0.0f;
        for (int i0 = 0; i0 < np; i0 += 64) {
            float wt = 0.0f;
            if (i0 + lane < np) {
                const float2 ml = *reinterpret_cast<const float2*>(piece(i0 + lane) + D);
                wt = ml.x == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(ml.x - mx);
                l += wt == 0.0f ? 0.0f : wt * ml.y;
            }
            const int m = min(64, np - i0);
#pragma unroll 8
            for (int i = 0; i < m; ++i) {
                const float wi = shfl(wt, i);
                const float* s = piece(i0 + i) + NPL * lane;
                float x[NPL];
                if constexpr (NPL == 1) x[0] = s[0];
                else {
                    const vec y = *reinterpret_cast<const vec*>(s);
#pragma unroll
                    for (int e = 0; e < NPL; ++e) x[e] = y[e];
                }
                // a piece of weight 0 adds nothing, not 0 * inf
#pragma unroll
                for (int e = 0; e < NPL; ++e) acc[e] = wi == 0.0f ? acc[e] : __builtin_fmaf(wi, x[e], acc[e]);
            }
        }
#pragma unroll
        for (int m = 32; m >= 1; m >>= 1) l += shfl_xor(l, m);
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        uint16_t* op = p.out + row * D + NPL * lane;
#pragma unroll
        for (int e = 0; e < NPL; ++e) op[e] = f32_to_half<BF>(acc[e] * inv);
    }
}

int launch_merge(const TileParams& p, int D, bool bf, int RB, hipStream_t s) {
    // a wave takes several rows where they are more than fill the chip
    const int64_t rows = (int64_t)p.total_rows * p.Hq;
    const int per = (int)((rows + 32767) / 32768);
    const dim3 grid((unsigned)((rows + 4 * per - 1) / (4 * per))), block(256);
    if (D == 64 && bf) hipLaunchKernelGGL((shared_merge_kernel<64, true>), grid, block, 0, s, p, RB, per);
    else if (D == 64) hipLaunchKernelGGL((shared_merge_kernel<64, false>), grid, block, 0, s, p, RB, per);
    else if (D == 128 && bf) hipLaunchKernelGGL((shared_merge_kernel<128, true>), grid, block, 0, s, p, RB, per);
    else if (D == 128) hipLaunchKernelGGL((shared_merge_kernel<128, false>), grid, block, 0, s, p, RB, per);
    else if (bf) hipLaunchKernelGGL((shared_merge_kernel<256, true>), grid, block, 0, s, p, RB, per);
    else hipLaunchKernelGGL((shared_merge_kernel<256, false>), grid, block, 0, s, p, RB, per);
    VMC_LAUNCH_CHECK();
    return VMC_OK;
}

// How a call runs, from its sizes alone (lengths are on the device).
struct Shape {
    int waves, whole, grid;  // waves of a workgroup; one item each; ranges (whole: workgroups)
    size_t cum, desc, gs, part, bytes;  // workspace offsets, size
};

Shape shape_of(bool paged, int rows, int nsets, int Hq, int Hkv, int D) {
    Shape sh = {};
    const int64_t G = Hq / Hkv;
    // workgroups that fit a CU: 64 KB of tiles each (head_dim 256: 128 KB)
    const int per_cu = D == 256 ? 1 : 2;
    sh.waves = 4;
    const int64_t items = (int64_t)Hkv * ((rows * G) / 256 + std::min(rows, nsets));
    // whole items of 256 rows where they are many times the CUs
    if (!paged && rows * G >= (int64_t)128 * nsets && items >= 4 * (int64_t)num_cus() && items < (1 << 30)) {
        sh.waves = 8;
        sh.whole = 1;
        sh.grid = (int)((items + 7) & ~7);
    } else {
        sh.grid = num_cus() * per_cu;
    }
    const int64_t total = paged ? (int64_t)nsets + rows : nsets;
    const int64_t RB = 32 * sh.waves;
    const int64_t prow = sh.whole ? 0 : paged ? sh.grid * RB + 2 * (int64_t)rows * Hq : 2 * sh.grid * RB;
    auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    sh.cum = 0;
    sh.desc = up((size_t)(total + 1) * sizeof(int64_t));
    sh.gs = sh.desc + up((size_t)total * sizeof(SetDesc));
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
    pl.RB = 32 * sh.waves;
    pl.paged = paged;
    pl.whole = sh.whole;
    pl.cum = reinterpret_cast<int64_t*>(w + sh.cum);
    pl.desc = reinterpret_cast<SetDesc*>(w + sh.desc);
    pl.gs = reinterpret_cast<int32_t*>(w + sh.gs);
    hipLaunchKernelGGL(shared_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, pl);
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
    p.gs = pl.gs;
    p.ns = a.nsets;
    p.nsets = pl.nsets;
    p.paged = paged;
    p.whole = sh.whole;
    p.total_rows = a.rows;
    p.grid = sh.grid;
    p.umin = 2;
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
    const int rc = a.D == 64    ? shared_tile_d64(p, src, bf, sh.waves, sh.grid, s)
                   : a.D == 128 ? shared_tile_d128(p, src, bf, sh.waves, sh.grid, s)
                                : shared_tile_d256(p, src, bf, sh.waves, sh.grid, s);
    if (rc != VMC_OK || sh.whole) return rc;
    return launch_merge(p, a.D, bf, pl.RB, s);
}

}  // namespace vmc
