// shared_tile.hpp -- the MFMA kernel of attention over keys that several rows share
// (shared_attn.hpp), for decode rows over a common prefix and over their own
// pages, and for decoder rows over an encoder's states.
//
// Work is a flat axis of units, a unit being one 64-key tile for one item; an
// item is a block of rows of one set and KV head.  All G query heads of a KV
// head share its keys, so a set's rows are its (token, head of the group)
// pairs: a group of 64 sequences with G = 4 fills 256 rows, a single sequence
// G of them.  Each workgroup takes one even range of the axis, whatever the
// sets' lengths are, and streams its tiles through LDS without a stop between
// items; a plan kernel turns the lengths into the axis (shared_plan.hip), and
// pieces of items that a range cut meet in a merge kernel through fp32 partial
// rows.  Where items are many times the workgroups (whole targets), each takes
// one whole item instead, without partial rows and merge.
//
// What bounds it: HBM with few rows, the matrix cores with many.
//   S^T[32 keys x 32 rows] = K . Q^T, O^T[D x 32 rows] += V^T . P^T on
//   v_mfma_f32_32x32x16: a row is one lane column in both, so its running max,
//   rescale and sums stay in the lane (and its partner 32 lanes on); V^T
//   operands come from the row-major tile by transposing LDS reads, and the
//   contraction index is permuted as P leaves the S registers (k = 8h + e <->
//   key 16c + 8 (e / 4) + 4h + e % 4).
//   A wave has 32 of the block's rows; waves beyond the rows only load.
// 16-bit rows arrive by load-to-LDS transfers, two or three tile slots; GGUF
// blocks through registers, dequantized to fp16 (code * d rounded once: 2^-11
// of a value at most).
//
// Weights enter P . V as two 16-bit terms of V's type, which leave 2^-17 (bf16)
// or 2^-23 (fp16) of a weight; one term would double the rounding error of the
// 16-bit result (its 2^-9 and the weights' 2^-9 in bf16).
#pragma once

#include "generic_row.hpp"
#include "kv_quant.hpp"
#include "prefill_dev.hpp"
#include "shared_plan.hpp"

namespace vmc {
namespace {

constexpr int kBN = 64;  // keys per tile

// two 16-bit terms of a pair of weights
template <bool BF>
__device__ __forceinline__ void two_terms(float a, float b, uint32_t& hi, uint32_t& lo) {
    hi = (uint32_t)f32_to_half<BF>(a) | ((uint32_t)f32_to_half<BF>(b) << 16);
    a -= half_to_f32<BF>((uint16_t)(hi & 0xffffu));
    b -= half_to_f32<BF>((uint16_t)(hi >> 16));
    lo = (uint32_t)f32_to_half<BF>(a) | ((uint32_t)f32_to_half<BF>(b) << 16);
}

// chunk swizzle of a tile row of 2 D bytes: 16-byte chunk ch of row r sits at
// ch ^ swz(r).  16 consecutive rows x one chunk (K operands) and 4 rows x 64
// bytes (transposing V reads) each cover the 64 banks once.
template <int D>
__device__ __forceinline__ int tile_swz(int r) {
    return D == 64 ? (((r >> 1) & 1) << 2) | ((r >> 2) & 3) : ((r & 3) << 2) | ((r >> 2) & 3);
}

enum { TS_LOCAL = 0, TS_PAGED = 1, TS_Q8 = 2, TS_Q4 = 3 };

// dma16s for a base that the compiler may have written by a vector instruction right
// before (a spilled SGPR read back by v_readlane): a vector memory access reads such
// an SGPR five wait states after the write at the earliest, and the compiler
// does not look into the asm.
__device__ __forceinline__ void dma16w(const void* base, uint32_t off, uint32_t m0) {
    asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "{m0}"(m0) : "memory");
}

template <typename T>
__device__ __forceinline__ const __attribute__((address_space(4))) T* as_const(const T* p) {
    return (const __attribute__((address_space(4))) T*)(uintptr_t)p;
}

// One row's keys k0 .. k1 - 1 by gen_row, from the head's rows at kp, vp (contiguous:
// of key 0; paged: of page 0, with the row's block table).  A call, not inlined:
// its registers stay out of the tile loop's, and its arguments are values, so
// that the kernel's parameters stay out of memory.
template <int D, int SRC, bool QBF>
__device__ __noinline__ void shared_row_exact(const uint16_t* q, const uint8_t* kp, const uint8_t* vp, int64_t k_row,
                                              int64_t v_row, const int32_t* bt, int64_t page_bytes, int bs, float scale,
                                              int k0, int k1, float* qs, uint16_t* out, float* part) {
    constexpr int GSRC = SRC == TS_LOCAL ? GEN_LOCAL : SRC == TS_Q8 ? GEN_Q8 : SRC == TS_Q4 ? GEN_Q4 : QBF ? GEN_BF16 : GEN_F16;
    const int lane = threadIdx.x & 63;
    GenArgs a = {};
    a.scale = scale;
    const TQTables none = {};
    wave_sync();
#pragma unroll
    for (int i = 0; i < D / 64; ++i) qs[lane + 64 * i] = half_to_f32<QBF>(q[lane + 64 * i]);
    wave_sync();
    auto key_at = [&](int k, const uint8_t*& ke, const uint8_t*& ve) __attribute__((always_inline)) {
        if constexpr (SRC == TS_LOCAL) {
            ke = kp + k * k_row;
            ve = vp + k * v_row;
            return true;
        } else {
            const int32_t id = bt[k / bs];
            const int64_t off = id * page_bytes + (int64_t)(k % bs) * k_row;
            ke = kp + off;
            ve = vp + off;
            return id >= 0;
        }
    };
    float m, l, acc[D / 64];
    gen_row<D, GSRC, 0, 0, QBF>(a, none, qs, lane, k0, k1, key_at, m, l, acc);
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
        if (out) out[lane + 64 * i] = f32_to_half<QBF>(acc[i] * inv);
        else part[lane + 64 * i] = acc[i];
    }
    if (!out && lane == 0) *reinterpret_cast<float2*>(part + D) = make_float2(m * kLog2e, l);
    wave_sync();
}

// BF: the products' type (LOCAL and PAGED: the rows'; GGUF: fp16, BF false);
// QBF: the type of q and out
template <int D, int SRC, bool QBF, int W>
__global__ void __launch_bounds__(64 * W, 2) shared_tile_kernel(TileParams p) {
    constexpr bool kGguf = SRC == TS_Q8 || SRC == TS_Q4;
    constexpr bool BF = QBF && !kGguf;
    using M = MT<BF>;
    using V8 = typename M::v8;
    constexpr int ROW = 2 * D, TILE = kBN * ROW;
    constexpr int NS = kGguf || D == 256 || (D == 128 && W == 4) ? 2 : 3;  // tile slots
    constexpr int NTR = TILE / (1024 * W);    // transfers per wave and tensor
    constexpr int HB = D == 256 ? 1 : 2;      // 32-key blocks per softmax round
    constexpr float kOff = BF ? 0.0f : 7.0f;  // weights are 2^(s - m + kOff), at most 2^15
    constexpr int RB = 32 * W;                // rows of an item
    // GGUF: blocks per lane and tile (K's then V's), dwords from a block's 4-byte floor
    constexpr int NBL = D / (16 * W) > 0 ? D / (16 * W) : 1;
    constexpr int BE = SRC == TS_Q8 ? 34 : 18, NWD = SRC == TS_Q8 ? 9 : 5;
    struct Lds {
        uint8_t tile[NS][2][TILE];  // [slot][K, V]
        float qs[W][D];             // rows that rerun key by key
    };
    __shared__ __attribute__((aligned(1024))) Lds lds;

    const int tid = threadIdx.x;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int c32 = lane & 31, h = lane >> 5;

    // ---- this workgroup's range of the axis
    int range;
    int64_t u0, u1;
    const int64_t total = as_const(p.cum)[p.nsets];
    if (p.whole) {  // one item; consecutive items to one XCD, whose L2 holds their keys
        const int64_t per = (total + 7) >> 3;
        range = (int)((blockIdx.x & 7) * per + (blockIdx.x >> 3));
        if ((blockIdx.x >> 3) >= per || range >= total) return;
        u0 = range;
        u1 = range + 1;
    } else {
        const int n = plan_ranges(total, p.grid, p.umin);
        range = n == p.grid && (n & 7) == 0 ? (int)((blockIdx.x & 7) * (n >> 3) + (blockIdx.x >> 3)) : (int)blockIdx.x;
        if (range >= n) return;
        u0 = range * total / n;
        u1 = (range + 1) * total / n;
        if (u0 >= u1) return;
    }
    struct Cursor {
        int set, g, rb, t;
        SetDesc d;
    };
    auto load_desc = [&](Cursor& c) __attribute__((always_inline)) {
        const auto* s = as_const(reinterpret_cast<const int*>(p.desc + c.set));
        c.d = SetDesc{s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7]};
    };
    auto advance = [&](Cursor& c) __attribute__((always_inline)) {
        if (++c.t < c.d.tiles) return;
        c.t = 0;
        if (++c.rb < c.d.nb) return;
        c.rb = 0;
        if (++c.g < p.Hkv) return;
        c.g = 0;
        do {
            if (++c.set >= p.nsets) return;  // past the axis: not used
            load_desc(c);
        } while (c.d.tiles == 0);
    };
    Cursor cc;
    cc.set = plan_find(p.cum, p.nsets, u0, lane);
    load_desc(cc);
    {
        const int64_t rem = u0 - as_const(p.cum)[cc.set];
        const int per = p.whole ? 1 : cc.d.tiles;
        const int item = (int)(rem / per);
        cc.t = (int)(rem % per);
        cc.g = item / cc.d.nb;
        cc.rb = item % cc.d.nb;
    }
    int units = p.whole ? cc.d.tiles : (int)(u1 - u0);  // to go
    Cursor pc = cc;

    // ---- fetch side.  A record names the tile to load next: base addresses of
    // this wave's rows (TS_LOCAL, TS_PAGED) or of the four pages
    const uint8_t *rk[kGguf ? 4 : 1], *rv[kGguf ? 4 : 1];
    int r_first = 0, r_last = 0;  // the wave's rows (GGUF: the tile's) clamp to these
    uint32_t r_valid = 0, vq = 0;  // 16-key chunks that hold keys: the record's, and those of loaded tiles
    auto fetch = [&]() __attribute__((always_inline)) {  // pc's tile
        const int k0 = (pc.d.klo & ~15) + kBN * pc.t, last = pc.d.khi - 1 - k0;
        const int first = max(pc.d.klo - k0, 0);
        if constexpr (SRC == TS_LOCAL) {
            const int64_t key = (int64_t)pc.d.src + k0;
            rk[0] = p.kp + key * p.k_row + pc.g * p.k_head;
            rv[0] = p.vp + key * p.v_row + pc.g * p.v_head;
            r_first = first;
            r_last = last;
            r_valid = (2u << min(3, last >> 4)) - 1u;
        } else {
            const auto* bt = as_const(p.bt + (int64_t)pc.d.src * p.max_blocks);
            int id[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int k = k0 + 16 * min(c, last >> 4);
                id[c] = bt[p.bs == 16 ? k >> 4 : k / p.bs];
            }
            r_valid = 0;
            int any = 0;  // a page for the rows of holes: their keys are masked, so it only has to be finite memory
#pragma unroll
            for (int c = 3; c >= 0; --c) {
                r_valid |= id[c] >= 0 && 16 * c <= last ? 1u << c : 0u;
                any = id[c] >= 0 ? id[c] : any;
            }
            r_first = first;
            r_last = last;
            auto at = [&](int c, int page, const uint8_t*& a, const uint8_t*& b) __attribute__((always_inline)) {
                const int k = k0 + 16 * min(c, last >> 4);
                const int in_page = p.bs == 16 ? 0 : k % p.bs;
                const int64_t off = (int64_t)(page >= 0 ? page : any) * p.page_bytes + (int64_t)in_page * p.k_row +
                                    pc.g * p.k_head;
                a = p.kp + off;
                b = p.vp + off;
            };
            if constexpr (kGguf) {
#pragma unroll
                for (int c = 0; c < 4; ++c) at(c, id[c], rk[c], rv[c]);
            } else {  // the wave's rows lie in one chunk
                const int c = 4 * w / W;
                int page = id[0];
#pragma unroll
                for (int i = 1; i < 4; ++i) page = c == i ? id[i] : page;
                at(c, page, rk[0], rv[0]);
            }
        }
    };
    // row r of the tile -> the row of its chunk to read (every row read is a key of the item)
    auto chunk_row = [&](int r) __attribute__((always_inline)) {
        const int c = min(r >> 4, r_last >> 4);
        const int x = c == (r_last >> 4) ? min(r & 15, r_last & 15) : (r & 15);
        return c == 0 ? max(x, r_first) : x;
    };
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(
        (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)&lds.tile[0][0][0]);
    uint32_t raw[kGguf ? NBL : 1][kGguf ? NWD : 1];
    auto load = [&](uint32_t slot) __attribute__((always_inline)) {  // the record's tile
        if constexpr (!kGguf) {
            const uint32_t dst = lds0 + slot * (2u * TILE) + 1024u * NTR * (uint32_t)w;
#pragma unroll
            for (int i = 0; i < NTR; ++i) {
                const int r = kBN / W * w + i * (1024 / ROW) + lane / (D / 8);
                const uint32_t col = 16u * (uint32_t)((lane % (D / 8)) ^ tile_swz<D>(r));
                uint32_t ko, vo;
                if constexpr (SRC == TS_LOCAL) {
                    const int x = max(min(r, r_last), r_first);
                    ko = (uint32_t)x * (uint32_t)p.k_row;
                    vo = (uint32_t)x * (uint32_t)p.v_row;
                } else {
                    ko = vo = (uint32_t)chunk_row(r) * (uint32_t)p.k_row;
                }
                dma16w(rk[0], ko + col, dst + 1024u * i);
                dma16w(rv[0], vo + col, dst + TILE + 1024u * i);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NBL; ++i) {
                const int idx = i * 64 * W + tid;
                if (NBL * 64 * W > 4 * D && idx >= 4 * D) break;
                const bool is_v = idx >= 2 * D;
                const int x = idx & (2 * D - 1), r = x / (D / 32), blk = x % (D / 32), c = r >> 4;
                const uint8_t* base = is_v ? rv[0] : rk[0];
#pragma unroll
                for (int e = 1; e < 4; ++e) base = c == e ? (is_v ? rv[e] : rk[e]) : base;
                // from the block's 4-byte floor: an odd block starts 2 bytes past one; the
                // last dword stays inside the entry
                const uint32_t* s = reinterpret_cast<const uint32_t*>(base + (uint32_t)chunk_row(r) * (uint32_t)p.k_row +
                                                                      BE * blk - 2 * (blk & 1));
                typedef uint32_t u32x4a __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll
                for (int e = 0; e + 4 <= NWD; e += 4) {
                    const u32x4a y = *reinterpret_cast<const u32x4a*>(s + e);
#pragma unroll
                    for (int j = 0; j < 4; ++j) raw[i][e + j] = y[j];
                }
                raw[i][NWD - 1] = s[NWD - 1];
            }
        }
    };
    auto stage = [&](uint32_t slot) __attribute__((always_inline)) {  // GGUF: registers -> tile
        if constexpr (kGguf) {
#pragma unroll
            for (int i = 0; i < NBL; ++i) {
                const int idx = i * 64 * W + tid;
                if (NBL * 64 * W > 4 * D && idx >= 4 * D) break;
                const int is_v = idx >= 2 * D;
                const int x = idx & (2 * D - 1), r = x / (D / 32), blk = x % (D / 32);
                const bool odd = (blk & 1) != 0;
                uint32_t c[NWD - 1];
#pragma unroll
                for (int e = 0; e < NWD - 1; ++e)
                    c[e] = odd ? raw[i][e + 1] : __builtin_amdgcn_alignbyte(raw[i][e + 1], raw[i][e], 2);
                const uint16_t db = (uint16_t)(odd ? raw[i][0] >> 16 : raw[i][0] & 0xffffu);
                const _Float16 dh = __builtin_bit_cast(_Float16, db);
                const f16x2 d2 = {dh, dh};
                uint8_t* row = lds.tile[slot][is_v] + r * ROW;
#pragma unroll
                for (int j = 0; j < 4; ++j) {  // chunk j: values 8j .. 8j + 7
                    u32x4 y;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if constexpr (SRC == TS_Q8)
                            y[e] = q8_pair_f16((e & 1) ? c[2 * j + e / 2] >> 16 : c[2 * j + e / 2] & 0xffffu, d2);
                        else
                            y[e] = q4_pair_f16((e & 1) ? c[2 * (j & 1) + e / 2] >> 16 : c[2 * (j & 1) + e / 2] & 0xffffu,
                                               j >= 2 ? 4 : 0, d2);
                    }
                    *reinterpret_cast<u32x4*>(row + 16 * ((4 * blk + j) ^ tile_swz<D>(r))) = y;
                }
            }
        }
    };

    // ---- compute side: operand addresses.  K: row 32 kb + c32, chunk 2s + h.  V
    // (transposing): lane (e, x) of a 16-lane group addresses 8 bytes of row e of
    // 4, and gets one dim of the 4 rows: dims 32 m + c32, keys 16 c + 8 sec + 4 h
    // + 0 .. 3
    const uint32_t k_lane = lds0 + (uint32_t)(c32 * ROW + 16 * (h ^ tile_swz<D>(c32)));
    const int te = (lane >> 2) & 3, tx = lane & 3, cb = (lane >> 4) & 1;
    uint32_t v_lane[2];
#pragma unroll
    for (int sec = 0; sec < 2; ++sec) {
        const int r = 8 * sec + 4 * h + te;
        v_lane[sec] = lds0 + TILE + (uint32_t)(r * ROW + 8 * (tx & 1) + 16 * ((2 * cb + (tx >> 1)) ^ tile_swz<D>(r)));
    }
    auto lds128 = [](uint32_t a) __attribute__((always_inline)) {
        return *reinterpret_cast<const __attribute__((address_space(3))) u32x4*>((uintptr_t)a);
    };
    auto lds_tr = [](uint32_t a) __attribute__((always_inline)) {
        return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                             (__attribute__((address_space(3))) s16x4*)(uintptr_t)a));
    };

    V8 qf[D / 16];
    f32x16 o[D / 32];
    // reference max (log2 units): moves only when a score passes it by more than 8
    float m_run = 0.f, m_thr = 0.f, l_part = 0.f, csc = 0.f;
    int lo = 0, hi = 0, hi_min = 0, nrow = 0;  // keys of this lane's row; the least hi of the wave; rows of the item
    int64_t tok = 0;
    int head = 0, seg_t0 = 0;
    bool row_ok = false, active = false;
    auto begin_item = [&]() __attribute__((always_inline)) {  // cc's, at tile cc.t
        const int all = cc.d.ntok * p.G;
        nrow = min(RB, all - RB * cc.rb);
        seg_t0 = cc.t;
        active = 32 * w < nrow;
        if (!active) return;
        const int r = RB * cc.rb + min(32 * w + c32, nrow - 1);
        row_ok = 32 * w + c32 < nrow;
        tok = cc.d.row0 + r / p.G;
        head = cc.g * p.G + r % p.G;
        lo = cc.d.klo;
        hi = cc.d.khi;
        if (SRC != TS_LOCAL && cc.d.own == 0) hi = min(hi, p.seq_lens[tok]);
        hi_min = hi;
        if (SRC != TS_LOCAL && cc.d.own == 0) {
#pragma unroll
            for (int m = 16; m >= 1; m >>= 1) hi_min = min(hi_min, __shfl_xor(hi_min, m, kWave));
            hi_min = __builtin_amdgcn_readfirstlane(hi_min);
        }
        const uint16_t* qp = p.q + tok * p.q_ts + head * p.q_hs + 8 * h;
        const float sl2 = p.scale * kLog2e;
        csc = fabsf(sl2);
        const uint32_t qflip = sl2 < 0.0f ? 0x80008000u : 0u;  // a negative scale flips Q's signs
        u32x4 x[D / 16];
#pragma unroll
        for (int s = 0; s < D / 16; ++s) x[s] = *reinterpret_cast<const u32x4*>(qp + 16 * s) ^ qflip;
        if constexpr (kGguf && QBF) {
            // bf16 q in fp16: the row scaled by a power of two so that its largest
            // value is in 2^7 .. 2^8, which csc undoes
            uint32_t mx = 0;
#pragma unroll
            for (int s = 0; s < D / 16; ++s)
#pragma unroll
                for (int e = 0; e < 4; ++e) mx = max(mx, max(x[s][e] & 0x7fffu, (x[s][e] >> 16) & 0x7fffu));
            mx = max(mx, (uint32_t)__shfl_xor((int)mx, 32, kWave));
            const int ex = min(max((int)(mx >> 7), 8), 254) - 127 - 7;  // biased exponent of the largest
            const float up = ldexpf(1.0f, -ex);
            csc = ldexpf(csc, ex);
#pragma unroll
            for (int s = 0; s < D / 16; ++s)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    x[s][e] = (uint32_t)f32_to_f16_bits(bf16_bits_to_f32((uint16_t)(x[s][e] & 0xffffu)) * up) |
                              ((uint32_t)f32_to_f16_bits(bf16_bits_to_f32((uint16_t)(x[s][e] >> 16)) * up) << 16);
        }
#pragma unroll
        for (int s = 0; s < D / 16; ++s) qf[s] = as_v8<V8>(x[s]);
#pragma unroll
        for (int m = 0; m < D / 32; ++m)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[m][i] = 0.0f;
        m_run = m_thr = -__builtin_inff();
        l_part = 0.0f;
    };

    auto process = [&](uint32_t slot, uint32_t valid) __attribute__((always_inline)) {
        const int kt = (cc.d.klo & ~15) + kBN * cc.t;
        const uint32_t k_slot = k_lane + slot * (2u * TILE);
        const uint32_t v_slot[2] = {v_lane[0] + slot * (2u * TILE), v_lane[1] + slot * (2u * TILE)};
#pragma unroll
        for (int r = 0; r < 2 / HB; ++r) {
            const int k0 = kt + 32 * HB * r;
            const uint32_t vb = HB == 2 ? valid : (valid >> (2 * r)) & 3u;
            if (vb == 0) continue;  // past the keys, or holes
            const bool need_mask = k0 + 32 * HB > hi_min || k0 < lo || vb != (HB == 2 ? 15u : 3u);
            f32x16 sacc[HB];
#pragma unroll
            for (int b = 0; b < HB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) sacc[b][i] = 0.0f;
            // K operands are read two steps ahead of their products, V operands one;
            // fixed by scheduling barriers, or the compiler issues each read right
            // before the product that waits for it
            constexpr int KA = 2, VA = 1;
            u32x4 ka[KA + 1][HB];
            auto read_k = [&](int s) __attribute__((always_inline)) {
#pragma unroll
                for (int b = 0; b < HB; ++b)
                    ka[s % (KA + 1)][b] = lds128((k_slot ^ (uint32_t)(32 * (s & 7))) +
                                                 (uint32_t)((HB * r + b) * 32 * ROW + 256 * (s >> 3)));
            };
#pragma unroll
            for (int s = 0; s < KA; ++s) read_k(s);
#pragma unroll
            for (int s = 0; s < D / 16; ++s) {
                if (s + KA < D / 16) read_k(s + KA);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int b = 0; b < HB; ++b) sacc[b] = M::mma(as_v8<V8>(ka[s % (KA + 1)][b]), qf[s], sacc[b]);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (need_mask) {
#pragma unroll
                for (int b = 0; b < HB; ++b)
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const int kv = k0 + 32 * b + 8 * (j >> 2) + 4 * h + (j & 3);
                        const bool there = ((vb >> (2 * b + (j >> 3))) & 1) != 0;
                        sacc[b][j] = kv < hi && kv >= lo && there ? sacc[b][j] : -__builtin_inff();
                    }
            }
            float mloc = sacc[0][0];
#pragma unroll
            for (int b = 0; b < HB; ++b)
#pragma unroll
                for (int j = 0; j < 16; ++j) mloc = fmaxf(mloc, sacc[b][j]);
            if (__ballot(mloc * csc > m_thr)) {  // rare after the first tiles
                const float mrow = fmaxf(mloc, shfl_xor(mloc, 32)) * csc;
                const bool upd = mrow > m_thr;  // the same in both halves of the row
                const float alpha = upd ? __builtin_amdgcn_exp2f(m_run - mrow) : 1.0f;  // 0 from -inf
                m_run = upd ? mrow : m_run;
                m_thr = m_run + 8.0f;
                l_part *= alpha;
#pragma unroll
                for (int m = 0; m < D / 32; ++m)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[m][i] *= alpha;
            }
            const float ref = m_run == -__builtin_inff() ? 0.0f : m_run - kOff;
            u32x4 pt[2][2 * HB];  // [term][16-key chunk]
            float sum = 0.0f;
#pragma unroll
            for (int c = 0; c < 2 * HB; ++c)
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const int j = 4 * (2 * (c & 1) + (e >> 2)) + (e & 3);
                    const float x0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[c >> 1][j], csc, -ref));
                    const float x1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[c >> 1][j + 1], csc, -ref));
                    sum += x0 + x1;
                    uint32_t t0, t1;
                    two_terms<BF>(x0, x1, t0, t1);
                    pt[0][c][e >> 1] = t0;
                    pt[1][c][e >> 1] = t1;
                }
            l_part += sum;
            u32x2 va[VA + 1][2];
            auto read_v = [&](int i) __attribute__((always_inline)) {
                const int c = i / (D / 32), m = i % (D / 32);
                const int vo = (2 * HB * r + c) * 16 * ROW + 256 * (m >> 2);
#pragma unroll
                for (int sec = 0; sec < 2; ++sec)
                    va[i % (VA + 1)][sec] = lds_tr((v_slot[sec] ^ (uint32_t)(64 * (m & 3))) + (uint32_t)vo);
            };
            constexpr int NV = 2 * HB * (D / 32);
#pragma unroll
            for (int i = 0; i < VA; ++i) read_v(i);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (i + VA < NV) read_v(i + VA);
                __builtin_amdgcn_sched_barrier(0);
                const int c = i / (D / 32), m = i % (D / 32);
                const u32x2* vi = va[i % (VA + 1)];
                const V8 x = as_v8<V8>(u32x4{vi[0][0], vi[0][1], vi[1][0], vi[1][1]});
#pragma unroll
                for (int u = 0; u < 2; ++u) o[m] = M::mma(x, as_v8<V8>(pt[u][c]), o[m]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };

    // ---- the segment of cc's item that ends after tile t_end - 1
    auto end_item = [&](int t_end) __attribute__((always_inline)) {
        const bool cut = seg_t0 > 0 || t_end < cc.d.tiles;
        // partial row 0 of the segment (shared_plan.hpp)
        const int64_t prow = p.paged ? plan_rows_paged(range, RB, p.Hq, p.G, p.total_rows, cc.d, cc.g, cc.rb)
                                     : plan_rows_local(range, RB, seg_t0 > 0);
        const bool direct = !p.paged && !cut;
        const float l = l_part + shfl_xor(l_part, 32);
        bool bad = !(l == l);
#pragma unroll
        for (int m = 0; m < D / 32; ++m)
#pragma unroll
            for (int i = 0; i < 16; ++i) bad |= !(fabsf(o[m][i]) < __builtin_inff());
        uint64_t badb = __ballot(bad && row_ok);
        badb = (badb | (badb >> 32)) & 0xffffffffull;  // a row is the lane and its partner
        if (row_ok && !((badb >> c32) & 1)) {
            if (direct) {
                const float inv = l > 0.0f ? 1.0f / l : 0.0f;
                uint16_t* op = p.out + (tok * p.Hq + head) * D + 4 * h;
#pragma unroll
                for (int m = 0; m < D / 32; ++m)
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        uint32_t x[2];
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            x[i] = (uint32_t)f32_to_half<QBF>(o[m][4 * b + 2 * i] * inv) |
                                   ((uint32_t)f32_to_half<QBF>(o[m][4 * b + 2 * i + 1] * inv) << 16);
                        *reinterpret_cast<u32x2*>(op + 32 * m + 8 * b) = u32x2{x[0], x[1]};
                    }
            } else {
                float* pp = p.part + (prow + 32 * w + c32) * (D + 4);
#pragma unroll
                for (int m = 0; m < D / 32; ++m)
#pragma unroll
                    for (int b = 0; b < 4; ++b)
                        *reinterpret_cast<f32x4*>(pp + 32 * m + 8 * b + 4 * h) =
                            f32x4{o[m][4 * b], o[m][4 * b + 1], o[m][4 * b + 2], o[m][4 * b + 3]};
                // o and l hold weights of 2^(s - m_run + kOff): the reference they go with
                if (h == 0) *reinterpret_cast<float2*>(pp + D) = make_float2(m_run - kOff, l);
            }
        }
        while (badb) {
            const int c = (int)__builtin_ctzll(badb);
            badb &= badb - 1;
            const int r = RB * cc.rb + 32 * w + c;
            const int64_t t = cc.d.row0 + r / p.G;
            const int hd = cc.g * p.G + r % p.G, kb = cc.d.klo & ~15;
            const int k0 = max(cc.d.klo, kb + kBN * seg_t0);
            const int k1 = min(__builtin_amdgcn_readlane(hi, c), kb + kBN * t_end);
            const int64_t koff = cc.g * p.k_head + (p.paged ? 0 : cc.d.src * p.k_row);
            const int64_t voff = cc.g * p.v_head + (p.paged ? 0 : cc.d.src * p.v_row);
            shared_row_exact<D, SRC, QBF>(p.q + t * p.q_ts + hd * p.q_hs, p.kp + koff, p.vp + voff, p.k_row, p.v_row,
                                          p.bt + (p.paged ? cc.d.src * p.max_blocks : 0), p.page_bytes, p.bs, p.scale,
                                          k0, k1, lds.qs[w],
                                          direct ? p.out + (t * p.Hq + hd) * D : nullptr,
                                          direct ? nullptr : p.part + (prow + 32 * w + c) * (D + 4));
        }
    };

    if (p.whole && units == 0) {  // rows of a sequence without states
        begin_item();
        if (active) {
#pragma unroll
            for (int m = 0; m < D / 32; ++m)
#pragma unroll
                for (int b = 0; b < 4; ++b)
                    if (row_ok)
                        *reinterpret_cast<u32x2*>(p.out + (tok * p.Hq + head) * D + 4 * h + 32 * m + 8 * b) = u32x2{0u, 0u};
        }
        return;
    }

    int fetched = 0, loaded = 0;  // tiles
    auto next_record = [&]() __attribute__((always_inline)) {
        if (fetched == units) return;
        if (fetched) advance(pc);
        fetch();
        ++fetched;
    };
    auto load_next = [&](uint32_t slot) __attribute__((always_inline)) {
        load(slot);
        vq = (vq << 4) | r_valid;
        ++loaded;
    };
    next_record();
    if constexpr (kGguf) {
        load_next(0);
        next_record();
        uint32_t slot = 0;
        for (int u = 0; u < units; ++u) {
            stage(slot);
            const uint32_t valid = vq & 15u;
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (loaded < units) {
                load_next(0);
                next_record();
            }
            if (u == 0 || cc.t == 0) begin_item();
            if (active) process(slot, valid);
            if (active && (cc.t + 1 == cc.d.tiles || u + 1 == units)) end_item(cc.t + 1);
            if (u + 1 < units) advance(cc);
            slot ^= 1;
        }
    } else {
        // tile u in slot u % NS, the next NS - 1 in flight while it runs.  The barrier
        // makes tile u visible and shows slot (u - 1) % NS free, which then receives
        // tile u + NS - 1 (2 NTR transfers a tile and wave; vmcnt retires in order)
        load_next(0);
        next_record();
        if (NS == 3 && loaded < units) {
            load_next(1);
            next_record();
        }
        uint32_t slot = 0, fill = NS - 1;
        for (int u = 0; u < units; ++u) {
            if (NS == 3 && loaded > u + 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * NTR) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (loaded < units) {
                load_next(fill);
                next_record();
            }
            if (u == 0 || cc.t == 0) begin_item();
            const uint32_t valid = (vq >> (4 * (loaded - u - 1))) & 15u;
            if (active) process(slot, valid);
            if (active && (cc.t + 1 == cc.d.tiles || u + 1 == units)) end_item(cc.t + 1);
            if (u + 1 < units) advance(cc);
            slot = slot == NS - 1 ? 0 : slot + 1;
            fill = fill == NS - 1 ? 0 : fill + 1;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
}

template <int D, int SRC, bool QBF, int W>
int launch_tile(const TileParams& p, unsigned grid, hipStream_t s) {
    hipLaunchKernelGGL((shared_tile_kernel<D, SRC, QBF, W>), dim3(grid), dim3(64 * W), 0, s, p);
    VMC_LAUNCH_CHECK();
    return VMC_OK;
}

template <int D>
int dispatch_tile(const TileParams& p, int src, bool qbf, int waves, unsigned grid, hipStream_t s) {
    switch (src) {
        case TS_LOCAL:
            if (waves == 8) return qbf ? launch_tile<D, TS_LOCAL, true, 8>(p, grid, s) : launch_tile<D, TS_LOCAL, false, 8>(p, grid, s);
            return qbf ? launch_tile<D, TS_LOCAL, true, 4>(p, grid, s) : launch_tile<D, TS_LOCAL, false, 4>(p, grid, s);
        case TS_PAGED: return qbf ? launch_tile<D, TS_PAGED, true, 4>(p, grid, s) : launch_tile<D, TS_PAGED, false, 4>(p, grid, s);
        case TS_Q8: return qbf ? launch_tile<D, TS_Q8, true, 4>(p, grid, s) : launch_tile<D, TS_Q8, false, 4>(p, grid, s);
        case TS_Q4: return qbf ? launch_tile<D, TS_Q4, true, 4>(p, grid, s) : launch_tile<D, TS_Q4, false, 4>(p, grid, s);
        default: return VMC_EINVAL;
    }
}

}  // namespace
}  // namespace vmc
