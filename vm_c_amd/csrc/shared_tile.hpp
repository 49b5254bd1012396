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
// items; a plan turns the lengths into the axis (shared_plan.hpp), and pieces of
// items that a range cut meet in a merge kernel through fp32 partial rows.
// Where items are many times the workgroups (whole targets), each takes one
// whole item instead, without partial rows and merge.
//
// What bounds it: HBM with few rows, with many the matrix cores together with the
// vector instructions of the softmax, which a wave's products wait for.
//   S^T[32 keys x 32 rows] = K . Q^T, O^T[D x 32 rows] += V^T . P^T on
//   v_mfma_f32_32x32x16: a row is one lane column in both, so its running max,
//   rescale and sums stay in the lane (and its partner 32 lanes on); V^T
//   operands come from the row-major tile by transposing LDS reads, and the
//   contraction index is permuted as P leaves the S registers (k = 8h + e <->
//   key 16c + 8 (e / 4) + 4h + e % 4).
//   A wave has 32 of the item's rows; waves beyond the rows only load.
// Measured (with the plan and merge): 32 sequences of 5 tokens, 200 to 4096 states, 32
// / 8 heads of 128, bf16: 47 us, 3.2 TB/s; 48 rows of head_dim 64 with 64 to 4096
// tokens of their own: 44 us, 2.6 TB/s; 64 rows over 32768 common tokens and 32 to
// 2048 own: 96 us, 2.7 TB/s and 0.36 PFLOP/s; 8 x 1024 rows over 2048 states: 360
// us, 0.76 PFLOP/s (a large product of the library: 1.21); 4 rows over 512 common
// tokens: 13.4 us, of which launch, plan and merge are 9.
//
// 16-bit rows arrive by load-to-LDS transfers, two or three tile slots; GGUF
// blocks through registers, dequantized to fp16 (code * d rounded once: 2^-11
// of a value at most) by two waves for the two that have rows.
//
// P . V runs in fp16.  A bf16 result takes weights of one fp16 term: two of them cut to
// fp16 by one instruction, and summed as they were cut by another, so that the cut (0
// to 2^-10 of a weight) stays out of their mean, and 2^-11 of a value at most is
// left, beside the result's own 2^-8 (two bf16 terms and bf16 V: 495 instead of 453 us
// for 8 x 1024 rows over 2048 states, the kernel alone, and no faster with few
// rows).  An fp16 result takes two terms, which leave 2^-23 of a weight: one would add
// as much error as the rounding of the result.
// bf16 V becomes fp16 in LDS, by the waves that fetched its rows, while slower waves
// still multiply: each 16 keys times 2^8 (values up to 255), 1 (larger ones) or
// 2^20 (all below 2^-12), which their weights undo against the largest of an
// item's.  So values from 2^-33 to 65504 keep their bits; the smaller ones of a
// chunk are cut, off by 2^-24 over its scale at most.  A chunk outside that range
// makes its rows rerun.
#pragma once

#include "generic_row.hpp"
#include "kv_quant.hpp"
#include "prefill_dev.hpp"
#include "shared_plan_dev.hpp"

namespace vmc {
namespace {

constexpr int kBN = 64;  // keys per tile

// two fp16 terms of a pair of weights
__device__ __forceinline__ void two_terms(float a, float b, uint32_t& hi, uint32_t& lo) {
    hi = (uint32_t)f32_to_half<false>(a) | ((uint32_t)f32_to_half<false>(b) << 16);
    a -= half_to_f32<false>((uint16_t)(hi & 0xffffu));
    b -= half_to_f32<false>((uint16_t)(hi >> 16));
    lo = (uint32_t)f32_to_half<false>(a) | ((uint32_t)f32_to_half<false>(b) << 16);
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

// QBF: the type of q and out (LOCAL and PAGED: of the rows too).  BF in it: K . Q runs in
// bf16 (GGUF: K is fp16 in LDS, and a bf16 q becomes it)
template <int D, int SRC, bool QBF>
__global__ void __launch_bounds__(256, tile_per_cu(D)) shared_tile_kernel(TileParams p) {
    constexpr int W = kTileWaves;
    constexpr bool kGguf = SRC == TS_Q8 || SRC == TS_Q4;
    constexpr bool BF = QBF && !kGguf;
    using M = MT<BF>;
    using V8 = typename M::v8;
    constexpr int ROW = 2 * D, TILE = kBN * ROW;
    constexpr int NS = kGguf || D != 64 ? 2 : 3;      // slots
    constexpr int NTR = TILE / (1024 * W);            // transfers per wave and tensor
    constexpr int CW = kGguf ? W / 2 : W;             // waves with rows; the others dequantize
    constexpr int RB = 32 * CW;                       // rows of an item
    constexpr bool kConv = BF;                        // bf16 V is converted to fp16
    constexpr int NT = QBF ? 1 : 2;                   // fp16 terms of a weight
    constexpr float kOff = 7.0f;                      // weights are 2^(s - m + kOff), at most 2^15
    constexpr int HB = D == 256 ? 1 : 2;              // 32-key blocks per softmax round
    // GGUF: blocks per dequantizing lane and tile (K's then V's), dwords from a block's
    // 4-byte floor
    constexpr int LOADERS = 64 * (W - CW), NBL = kGguf ? 4 * D / (kGguf ? LOADERS : 1) : 1;
    constexpr int BE = SRC == TS_Q8 ? 34 : 18, NWD = SRC == TS_Q8 ? 9 : 5;
    struct Lds {
        uint8_t tile[NS][2][TILE];                       // [slot][K, V]
        float qs[W][D];                                  // rows that rerun key by key
        alignas(16) SetDesc desc[kPlanFused];            // (fused)
        float vexp[2][W];                                // kConv [tile][16-key chunk]: 8 - log2 of V's scale
    };
    __shared__ __attribute__((aligned(1024))) Lds lds;

    const int tid = threadIdx.x;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int c32 = lane & 31, h = lane >> 5;

    // The parameters as rare steps read them: from the kernel's arguments in memory, there
    // and then, as the compiler would otherwise keep each in scalar registers from
    // the start and spill those (to vector lanes, read back in every tile)
    auto arg = [&]() __attribute__((always_inline)) {
        auto a = (const __attribute__((address_space(4))) TileParams*)__builtin_amdgcn_kernarg_segment_ptr();
        asm volatile("" : "+s"(a));
        return a;
    };
    // ---- this workgroup's tiles.  Of a set, a cursor keeps what each tile needs; the rest
    // is read again (through the scalar cache) where an item begins or ends.
    struct Cursor {
        int set, g, rb, t, tiles, nb, klo, khi, src;
    };
    auto uniform = [](const SetDesc& d) __attribute__((always_inline)) {
        auto f = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
        return SetDesc{f(d.row0), f(d.ntok), f(d.klo), f(d.khi), f(d.src), f(d.nb), f(d.tiles), f(d.own)};
    };
    auto desc_of = [&](int set) __attribute__((always_inline)) {
        if (arg()->fused) return uniform(lds.desc[set]);
        const auto* s = as_const(reinterpret_cast<const int*>(arg()->desc + set));
        return SetDesc{s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7]};
    };
    auto take = [&](Cursor& c, const SetDesc& d) __attribute__((always_inline)) {
        c.tiles = d.tiles;
        c.nb = d.nb;
        c.klo = d.klo;
        c.khi = d.khi;
        c.src = d.src;
    };
    auto advance = [&](Cursor& c) __attribute__((always_inline)) {
        if (++c.t < c.tiles) return;
        c.t = 0;
        if (++c.rb < c.nb) return;
        c.rb = 0;
        if (++c.g < arg()->Hkv) return;
        c.g = 0;
        do {
            if (++c.set >= arg()->nsets) return;  // past the axis: not used
            take(c, desc_of(c.set));
        } while (c.tiles == 0);
    };
    Cursor cc;  // of the tile in use
    int range = blockIdx.x, units;
    SetDesc first;
    using Plan = PlanLds<kPlanFused, W>;
    static_assert(sizeof(Plan) <= sizeof(lds.tile), "the plan's sums lie where tiles will");
    Plan& plan = *reinterpret_cast<Plan*>(&lds.tile[0][0][0]);
    if (p.whole) {  // one item; consecutive items to one XCD, whose L2 holds their keys
        const int64_t total = as_const(p.cum)[p.nsets], per = (total + 7) >> 3;
        const int64_t item = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
        if ((blockIdx.x >> 3) >= per || item >= total) return;
        cc.set = plan_find(p.cum, p.nsets, item, lane);
        first = desc_of(cc.set);
        take(cc, first);
        const int in_set = (int)(item - as_const(p.cum)[cc.set]);
        cc.t = 0;
        cc.g = in_set / cc.nb;
        cc.rb = in_set % cc.nb;
        units = cc.tiles;
    } else if (p.fused) {
        const PlanSums sums = plan_sets(p.plan, plan, lds.desc, tid);
        if (blockIdx.x == 0) plan_out(p.plan, sums, lds.desc, plan.cum, tid);
        RangeRec r = {};
        const int n = plan_ranges(sums.total, p.grid, p.cus);
        if (range < n) {  // even lanes: where the range begins, odd ones: where the next does
            const int u = (int)div_floor<long long>((long long)(range + (lane & 1)) * sums.total, n);
            const int before = u < sums.total ? range_begin(plan, lds.desc, p.nsets, u, r) : sums.total_t;
            r.ntiles = __builtin_amdgcn_readlane(before, 1) - __builtin_amdgcn_readlane(before, 0);
        }
        if (tid == 0 && !p.paged) const_cast<RangeRec*>(p.range)[range] = r;  // (the merge's)
        cc.set = __builtin_amdgcn_readfirstlane(r.set);
        cc.g = __builtin_amdgcn_readfirstlane(r.g);
        cc.rb = __builtin_amdgcn_readfirstlane(r.rb);
        cc.t = __builtin_amdgcn_readfirstlane(r.t);
        units = __builtin_amdgcn_readfirstlane(r.ntiles);
        first = uniform(r.d);
        take(cc, first);
        if (units == 0) return;
        __syncthreads();  // the plan's sums are read
    } else {
        const auto* r = as_const(reinterpret_cast<const int*>(p.range + range));
        cc.set = r[0];
        cc.g = r[1];
        cc.rb = r[2];
        cc.t = r[3];
        units = r[4];
        first = SetDesc{r[8], r[9], r[10], r[11], r[12], r[13], r[14], r[15]};
        take(cc, first);
        if (units == 0) return;
    }
    units = __builtin_amdgcn_readfirstlane(units);

    // ---- fetch side.  A record names a tile's memory: the offset of this wave's rows
    // (TS_LOCAL, TS_PAGED) or of the four 16-key chunks (GGUF), and the rows that all
    // others clamp to, so that each row read is a key of the item
    constexpr int NA = kGguf ? 4 : 1;
    struct Rec {
        int64_t k[NA], v;  // (paged: k for both)
        int first, last;
    };
    Cursor pc = cc;
    Rec rec;            // of the next tile to load
    uint32_t vq = 0;    // 16-key chunks that hold keys, 4 bits a tile, the latest fetched lowest
    int fetched = 0;    // tiles with a record
    auto fetch = [&]() __attribute__((always_inline)) {
        if (fetched == units) return;
        if (fetched) advance(pc);
        ++fetched;
        const int k0 = (pc.klo & ~15) + kBN * pc.t, last = pc.khi - 1 - k0;
        rec.first = max(pc.klo - k0, 0);
        rec.last = last;
        if constexpr (SRC == TS_LOCAL) {
            const int64_t key = (int64_t)pc.src + k0;
            rec.k[0] = key * p.k_row + pc.g * p.k_head;
            rec.v = key * p.v_row + pc.g * p.v_head;
            vq = (vq << 4) | ((2u << min(3, last >> 4)) - 1u);
        } else {
            const auto* bt = as_const(p.bt + (int64_t)pc.src * p.max_blocks);
            int id[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int k = k0 + 16 * min(c, last >> 4);
                id[c] = bt[p.bs == 16 ? k >> 4 : k / p.bs];
            }
            uint32_t valid = 0;
            int any = 0;  // a page for the rows of holes: their keys are masked
#pragma unroll
            for (int c = 3; c >= 0; --c) {
                valid |= id[c] >= 0 && 16 * c <= last ? 1u << c : 0u;
                any = id[c] >= 0 ? id[c] : any;
            }
            vq = (vq << 4) | valid;
            auto at = [&](int c, int page) __attribute__((always_inline)) {
                const int k = k0 + 16 * min(c, last >> 4);
                const int in_page = p.bs == 16 ? 0 : k % p.bs;
                return (int64_t)(page >= 0 ? page : any) * p.page_bytes + (int64_t)in_page * p.k_row + pc.g * p.k_head;
            };
            if constexpr (kGguf) {
#pragma unroll
                for (int c = 0; c < 4; ++c) rec.k[c] = at(c, id[c]);
            } else {  // the wave's rows lie in one chunk
                const int c = 4 * w / W;
                int page = id[0];
#pragma unroll
                for (int i = 1; i < 4; ++i) page = c == i ? id[i] : page;
                rec.k[0] = at(c, page);
            }
        }
    };
    // row r of a tile -> the row of its 16-key chunk to read
    auto chunk_row = [&](int r, const Rec& x) __attribute__((always_inline)) {
        const int c = min(r >> 4, x.last >> 4);
        const int y = c == (x.last >> 4) ? min(r & 15, x.last & 15) : (r & 15);
        return c == 0 ? max(y, x.first) : y;
    };
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(
        (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)&lds.tile[0][0][0]);
    // Row of the tile that transfer i of this wave brings to this lane, and its bytes' place
    // in the row: the swizzle of rows TR i and the lane's own have no bit in common
    constexpr int TR = 1024 / ROW;
    int lane_row = lane / (D / 8);
    uint32_t lane_col = 16u * (uint32_t)((lane % (D / 8)) ^ tile_swz<D>(lane_row));
    auto part_row = [&](int i) __attribute__((always_inline)) { return kBN / W * w + TR * i + lane_row; };
    auto part_col = [&](int i) __attribute__((always_inline)) { return lane_col ^ (16u * (uint32_t)tile_swz<D>(TR * i)); };
    // (paged: of the row in its 16-key chunk, the same for K and V)
    uint32_t off_k = (uint32_t)part_row(0) % (SRC == TS_LOCAL ? kBN : 16) * (uint32_t)p.k_row;
    uint32_t off_v = SRC == TS_LOCAL ? (uint32_t)part_row(0) * (uint32_t)p.v_row : off_k;
    // this wave's part of K or V of a tile into LDS at dst
    auto transfer = [&](bool is_v, const Rec& x, uint32_t dst) __attribute__((always_inline)) {
        const uint64_t b64 = (uint64_t)(is_v ? p.vp + (SRC == TS_LOCAL ? x.v : x.k[0]) : p.kp + x.k[0]);
        const uint8_t* base = (const uint8_t*)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(b64 >> 32)) << 32) |
                                               (uint32_t)__builtin_amdgcn_readfirstlane((int)b64));
        const bool own_v = SRC == TS_LOCAL && is_v;
        dst += 1024u * NTR * (uint32_t)w;
        const uint32_t step = (uint32_t)(own_v ? p.v_row : p.k_row);
        // opaque, or the compiler computes every transfer's offset ahead, and where those fill
        // the registers (head_dim 256) reads them from memory between transfers, behind a
        // wait for all of them
        if constexpr (D == 256) asm volatile("" : "+v"(lane_row), "+v"(lane_col), "+v"(off_k), "+v"(off_v));
        if (x.first == 0 && x.last >= kBN - 1) {
#pragma unroll
            for (int i = 0; i < NTR; ++i)
                dma16w(base, (own_v ? off_v : off_k) + TR * i * step + part_col(i), dst + 1024u * i);
            return;
        }
#pragma unroll
        for (int i = 0; i < NTR; ++i) {
            const int r = part_row(i);
            const int y = SRC == TS_LOCAL ? max(min(r, x.last), x.first) : chunk_row(r, x);
            dma16w(base, (uint32_t)y * step + part_col(i), dst + 1024u * i);
        }
    };
    uint32_t blk_raw[kGguf ? NBL : 1][kGguf ? NWD : 1];
    auto load_blocks = [&]() __attribute__((always_inline)) {  // GGUF: the record's tile into registers
        if constexpr (kGguf) {
#pragma unroll
            for (int i = 0; i < NBL; ++i) {
                const int idx = i * LOADERS + tid - 64 * CW;
                const bool is_v = idx >= 2 * D;
                const int x = idx & (2 * D - 1), r = x / (D / 32), blk = x % (D / 32), c = r >> 4;
                int64_t off = rec.k[0];
#pragma unroll
                for (int e = 1; e < NA; ++e) off = c == e ? rec.k[e] : off;
                // from the block's 4-byte floor: an odd block starts 2 bytes past one; the
                // last dword stays inside the entry
                const uint32_t row = (uint32_t)chunk_row(r, rec);
                const uint32_t* s = reinterpret_cast<const uint32_t*>((is_v ? p.vp : p.kp) + off + row * (uint32_t)p.k_row +
                                                                      BE * blk - 2 * (blk & 1));
                typedef uint32_t u32x4a __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll
                for (int e = 0; e + 4 <= NWD; e += 4) {
                    const u32x4a y = *reinterpret_cast<const u32x4a*>(s + e);
#pragma unroll
                    for (int j = 0; j < 4; ++j) blk_raw[i][e + j] = y[j];
                }
                blk_raw[i][NWD - 1] = s[NWD - 1];
            }
        }
    };
    auto stage = [&](uint32_t slot) __attribute__((always_inline)) {  // GGUF: registers -> tile
        if constexpr (kGguf) {
#pragma unroll
            for (int i = 0; i < NBL; ++i) {
                const int idx = i * LOADERS + tid - 64 * CW;
                const bool is_v = idx >= 2 * D;
                const int x = idx & (2 * D - 1), r = x / (D / 32), blk = x % (D / 32);
                const bool odd = (blk & 1) != 0;
                uint32_t c[NWD - 1];
#pragma unroll
                for (int e = 0; e < NWD - 1; ++e)
                    c[e] = odd ? blk_raw[i][e + 1] : __builtin_amdgcn_alignbyte(blk_raw[i][e + 1], blk_raw[i][e], 2);
                const uint16_t db = (uint16_t)(odd ? blk_raw[i][0] >> 16 : blk_raw[i][0] & 0xffffu);
                const _Float16 dh = __builtin_bit_cast(_Float16, db);
                const f16x2 d2 = {dh, dh};
                uint8_t* row = lds.tile[slot][is_v ? 1 : 0] + r * ROW;
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
    // The V rows that this wave fetched of the tile in `slot`, one 16-key chunk, to fp16
    auto convert = [&](uint32_t slot, int half) __attribute__((always_inline)) {
        if constexpr (kConv) {
            typedef uint16_t u16x2v __attribute__((ext_vector_type(2)));
            uint32_t mx = 0;  // packed 16-bit maxima of the magnitudes
            uint8_t* at = lds.tile[slot][1] + 1024u * NTR * (uint32_t)w + 16u * (uint32_t)lane;
            u32x4 x[NTR];
#pragma unroll
            for (int i = 0; i < NTR; ++i) {
                x[i] = *reinterpret_cast<const u32x4*>(at + 1024 * i);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    mx = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2v, mx),
                                                                                __builtin_bit_cast(u16x2v, x[i][e] & 0x7fff7fffu)));
            }
            const uint32_t m = max(mx & 0xffffu, mx >> 16);
            // 2^8 for values up to 255, 1 for larger ones, 2^20 where all are below 2^-12
            const bool big = __ballot(m >= 0x4380u) != 0, tiny = __ballot(m >= 0x3980u) == 0;
            // past 65504 (or no number), or all below 2^-33 but not 0: no scale fits
            const bool bad = __ballot(m >= 0x4780u) != 0 || (__ballot(m >= 0x2f00u) == 0 && __ballot(m != 0) != 0);
            // (added to the exponents; a 0 becomes a number below fp16's, cut to 0 again)
            const uint32_t up = big ? 0u : tiny ? 20u << 23 : 8u << 23;
            if (lane == 0) lds.vexp[half][w] = bad ? __builtin_nanf("") : big ? 8.0f : tiny ? -12.0f : 0.0f;
#pragma unroll
            for (int i = 0; i < NTR; ++i) {
                u32x4 y;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t f0 = (x[i][e] << 16) + up, f1 = (x[i][e] & 0xffff0000u) + up;
                    y[e] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(__builtin_bit_cast(float, f0),
                                                                                   __builtin_bit_cast(float, f1)));
                }
                *reinterpret_cast<u32x4*>(at + 1024 * i) = y;
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
    float v_base = 0.f;  // kConv: the largest vexp so far; o is 2^(8 - v_base) times the sums
    int lo = 0, hi = 0, hi_min = 0;  // keys of this lane's row, the least end of the wave's rows
    bool active = false;             // the wave has rows of the item

    auto begin_item = [&](const SetDesc& d) __attribute__((always_inline)) {  // cc's, of set d
        const auto* a = arg();
        const int G = a->G, nrow = min(RB, d.ntok * G - RB * cc.rb);
        active = w < CW && 32 * w < nrow;
        if (!active) return;
        const int r = RB * cc.rb + min(32 * w + c32, nrow - 1);
        const int64_t tok = d.row0 + r / G;
        const uint16_t* qp = a->q + tok * a->q_ts + (cc.g * G + r % G) * a->q_hs + 8 * h;
        u32x4 x[D / 16];
#pragma unroll
        for (int s = 0; s < D / 16; ++s) x[s] = *reinterpret_cast<const u32x4*>(qp + 16 * s);
        lo = d.klo;
        hi = hi_min = d.khi;
        if (SRC != TS_LOCAL && d.own == 0) {
            hi = min(hi, a->seq_lens[tok]);
            hi_min = hi;
#pragma unroll
            for (int m = 16; m >= 1; m >>= 1) hi_min = min(hi_min, __shfl_xor(hi_min, m, kWave));
            hi_min = __builtin_amdgcn_readfirstlane(hi_min);
        }
        const float sl2 = a->scale * kLog2e;
        csc = fabsf(sl2);
        if (sl2 < 0.0f) {  // a negative scale flips Q's signs
#pragma unroll
            for (int s = 0; s < D / 16; ++s) x[s] ^= 0x80008000u;
        }
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
        // waited for here, before more transfers are issued: the compiler would wait for
        // those too
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
            asm volatile("" : "+v"(x[s]));
            qf[s] = as_v8<V8>(x[s]);
        }
#pragma unroll
        for (int m = 0; m < D / 32; ++m)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[m][i] = 0.0f;
        m_run = m_thr = v_base = -__builtin_inff();
        l_part = 0.0f;
    };

    // the tile in `slot`; valid: its 16-key chunks that hold keys; vexp: what weights of a
    // chunk are scaled by, as powers of two (kConv)
    auto process = [&](uint32_t slot, uint32_t valid, f32x4 vexp) __attribute__((always_inline)) {
        const int kt = (cc.klo & ~15) + kBN * cc.t;
        const uint32_t k_slot = k_lane + slot * (2u * TILE);
        const uint32_t vbase[2] = {v_lane[0] + slot * (2u * TILE), v_lane[1] + slot * (2u * TILE)};
#pragma unroll
        for (int r = 0; r < 2 / HB; ++r) {
            const int k0 = kt + 32 * HB * r;
            const uint32_t vb = HB == 2 ? valid : (valid >> (2 * r)) & 3u;
            if (vb == 0) continue;  // past the keys, or holes
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
            if (k0 + 32 * HB > hi_min || k0 < lo || vb != (HB == 2 ? 15u : 3u)) {
                asm volatile("");  // a branch: most tiles need none of this
                const int up = hi - k0 - 4 * h, dn = lo - k0 - 4 * h;
#pragma unroll
                for (int b = 0; b < HB; ++b)
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const int x = 32 * b + 8 * (j >> 2) + (j & 3);
                        const bool there = ((vb >> (2 * b + (j >> 3))) & 1) != 0;
                        sacc[b][j] = x < up && x >= dn && there ? sacc[b][j] : -__builtin_inff();
                    }
            }
            float mloc = sacc[0][0];
#pragma unroll
            for (int b = 0; b < HB; ++b)
#pragma unroll
                for (int j = 0; j < 16; ++j) mloc = fmaxf(mloc, sacc[b][j]);
            float top = v_base;  // kConv: of the largest values so far
            if constexpr (kConv) top = fmaxf(top, fmaxf(fmaxf(vexp[0], vexp[1]), fmaxf(vexp[2], vexp[3])));
            if (__ballot(mloc * csc > m_thr || top > v_base)) {  // rare after the first tiles
                const float mrow = fmaxf(mloc, shfl_xor(mloc, 32)) * csc;
                const bool upd = mrow > m_thr;  // the same in both halves of the row
                float alpha = upd ? __builtin_amdgcn_exp2f(m_run - mrow) : 1.0f;  // 0 from -inf
                m_run = upd ? mrow : m_run;
                m_thr = m_run + 8.0f;
                l_part *= alpha;
                if constexpr (kConv) alpha *= __builtin_amdgcn_exp2f(v_base - top);  // 0 from -inf
                v_base = top;
#pragma unroll
                for (int m = 0; m < D / 32; ++m)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[m][i] *= alpha;
            }
            const float ref = m_run == -__builtin_inff() ? 0.0f : m_run - kOff;
            u32x4 pt[2][2 * HB];  // [term][16-key chunk]
            float sum = 0.0f;
#pragma unroll
            for (int c = 0; c < 2 * HB; ++c) {
                const float off = kConv ? (vexp[2 * HB * r + c] - v_base) - ref : -ref;
                float part = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const int j = 4 * (2 * (c & 1) + (e >> 2)) + (e & 3);
                    const float x0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[c >> 1][j], csc, off));
                    const float x1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[c >> 1][j + 1], csc, off));
                    if constexpr (NT == 1) {
                        const auto xh = __builtin_amdgcn_cvt_pkrtz(x0, x1);
                        part = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, xh), f16x2{1, 1}, part, false);
                        pt[0][c][e >> 1] = __builtin_bit_cast(uint32_t, xh);
                    } else {
                        part += x0 + x1;
                        uint32_t t0, t1;
                        two_terms(x0, x1, t0, t1);
                        pt[0][c][e >> 1] = t0;
                        pt[1][c][e >> 1] = t1;
                    }
                }
                sum += kConv ? part * __builtin_amdgcn_exp2f(v_base - vexp[2 * HB * r + c]) : part;
            }
            // O^T += V^T P^T
            using MP = MT<false>;
            using VP = typename MP::v8;
            u32x2 va[VA + 1][2];
            auto read_v = [&](int i) __attribute__((always_inline)) {
                const int c = i / (D / 32), m = i % (D / 32);
                const int vo = (2 * HB * r + c) * 16 * ROW + 256 * (m >> 2);
#pragma unroll
                for (int sec = 0; sec < 2; ++sec)
                    va[i % (VA + 1)][sec] = lds_tr((vbase[sec] ^ (uint32_t)(64 * (m & 3))) + (uint32_t)vo);
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
                const VP x = as_v8<VP>(u32x4{vi[0][0], vi[0][1], vi[1][0], vi[1][1]});
#pragma unroll
                for (int u = 0; u < NT; ++u) o[m] = MP::mma(x, as_v8<VP>(pt[u][c]), o[m]);
                __builtin_amdgcn_sched_barrier(0);
            }
            l_part += sum;
        }
    };

    bool bad_seen = false;
    // ---- the segment (tiles t0 .. t1 - 1) of item (set, g, rb) ends
    auto end_item = [&](int set, int g, int rb, int t0, int t1) __attribute__((always_inline)) {
        const auto* a = arg();
        const SetDesc d = desc_of(set);
        const int G = a->G, nrow = min(RB, d.ntok * G - RB * rb);
        const bool row_ok = 32 * w + c32 < nrow;
        const bool cut = t0 > 0 || t1 < d.tiles;
        // partial row 0 of the segment (shared_plan.hpp)
        const int64_t prow = a->paged ? plan_rows_paged(range, RB, a->Hq, G, a->total_rows, d.own, d.row0, d.ntok, g, rb)
                                      : plan_rows_local(range, RB, t0 > 0);
        const bool direct = !a->paged && !cut;
        const float l = l_part + shfl_xor(l_part, 32);
        bool bad = !(l == l);
#pragma unroll
        for (int m = 0; m < D / 32; ++m)
#pragma unroll
            for (int i = 0; i < 16; ++i) bad |= !(fabsf(o[m][i]) < __builtin_inff());
        bad_seen |= __ballot(bad && row_ok) != 0;
        if (!row_ok) return;
        const float vs = kConv ? __builtin_amdgcn_exp2f(v_base - 8.0f) : 1.0f;
        if (direct) {
            const int r = RB * rb + 32 * w + c32;
            const float inv = l > 0.0f ? vs / l : 0.0f;
            uint16_t* op = a->out + ((int64_t)(d.row0 + r / G) * a->Hq + g * G + r % G) * D + 4 * h;
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
            float* pp = a->part + (prow + 32 * w + c32) * (D + 4);
#pragma unroll
            for (int m = 0; m < D / 32; ++m)
#pragma unroll
                for (int b = 0; b < 4; ++b)
                    *reinterpret_cast<f32x4*>(pp + 32 * m + 8 * b + 4 * h) =
                        f32x4{o[m][4 * b], o[m][4 * b + 1], o[m][4 * b + 2], o[m][4 * b + 3]} * vs;
            // o and l hold weights of 2^(s - m_run + kOff): the reference they go with
            if (h == 0) *reinterpret_cast<float2*>(pp + D) = make_float2(m_run - kOff, l);
        }
    };
    // Rows whose sums met an infinity or a NaN (a product takes every key's V times its
    // weight, also where that is 0) go key by key.  After the range, so that the
    // call has nothing of the loop's to keep: its segments are walked again, and the
    // rows in question known by what was written
    auto rerun = [&](Cursor c, int n) __attribute__((always_inline)) {
        const auto* a = arg();
        while (n > 0) {
            const SetDesc d = desc_of(c.set);
            const int G = a->G, nrow = min(RB, d.ntok * G - RB * c.rb), t0 = c.t, t1 = min(d.tiles, t0 + n);
            const bool direct = !a->paged && t0 == 0 && t1 == d.tiles;
            const int64_t prow = a->paged ? plan_rows_paged(range, RB, a->Hq, G, a->total_rows, d.own, d.row0, d.ntok, c.g, c.rb)
                                          : plan_rows_local(range, RB, t0 > 0);
            for (int i = 32 * w; i < min(32 * w + 32, nrow); ++i) {
                const int r = RB * c.rb + i, hd = c.g * G + r % G, kb = d.klo & ~15;
                const int64_t t = d.row0 + r / G;
                uint16_t* op = a->out + (t * a->Hq + hd) * D;
                float* pp = a->part + (prow + i) * (D + 4);
                bool bad = false;
#pragma unroll
                for (int k = 0; k < D / 64; ++k) {
                    const float x = direct ? half_to_f32<QBF>(__builtin_nontemporal_load(op + lane + 64 * k))
                                           : __builtin_nontemporal_load(pp + lane + 64 * k);
                    bad |= !(fabsf(x) < __builtin_inff());
                }
                if (!direct) bad |= !(__builtin_nontemporal_load(pp + D + 1) < __builtin_inff());
                if (__ballot(bad) == 0) continue;
                int k1 = min(d.khi, kb + kBN * t1);
                if (SRC != TS_LOCAL && d.own == 0) k1 = min(k1, a->seq_lens[t]);
                const int64_t koff = c.g * a->k_head + (a->paged ? 0 : d.src * a->k_row);
                const int64_t voff = c.g * a->v_head + (a->paged ? 0 : d.src * a->v_row);
                shared_row_exact<D, SRC, QBF>(a->q + t * a->q_ts + hd * a->q_hs, a->kp + koff, a->vp + voff, a->k_row,
                                              a->v_row, a->bt + (a->paged ? d.src * a->max_blocks : 0), a->page_bytes,
                                              a->bs, a->scale, max(d.klo, kb + kBN * t0), k1, lds.qs[w],
                                              direct ? op : nullptr, direct ? nullptr : pp);
            }
            n -= t1 - t0;
            if (n <= 0) break;
            c.t = d.tiles - 1;
            c.tiles = d.tiles;
            advance(c);
        }
    };

    if (units == 0) {  // (whole items) rows of a sequence without states
        const auto* a = arg();
        const SetDesc d = desc_of(cc.set);
        const int nrow = min(RB, d.ntok * a->G - RB * cc.rb);
        for (int i = tid; i < nrow * (D / 8); i += 64 * W) {
            const int r = RB * cc.rb + i / (D / 8);
            *reinterpret_cast<u32x4*>(a->out + ((int64_t)(d.row0 + r / a->G) * a->Hq + cc.g * a->G + r % a->G) * D +
                                      8 * (i % (D / 8))) = u32x4{0u, 0u, 0u, 0u};
        }
        return;
    }

    const Cursor start = cc;
    int loaded = 0, seg_t0 = cc.t;
    auto load = [&](uint32_t slot) __attribute__((always_inline)) {  // the record's tile
        if constexpr (kGguf) {
            load_blocks();  // into registers
        } else {
            transfer(false, rec, lds0 + slot * (2u * TILE));
            transfer(true, rec, lds0 + slot * (2u * TILE) + TILE);
        }
        ++loaded;
        fetch();
    };
    auto landed = [&](int u) __attribute__((always_inline)) {  // this wave's part of tile u
        if constexpr (!kGguf) {  // (vmcnt retires in order)
            if (NS == 3 && loaded > u + 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * NTR) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
    };
    auto meet = [&]() __attribute__((always_inline)) { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    // tile u by the waves that have rows
    auto use = [&](int u, uint32_t slot) __attribute__((always_inline)) {
        const uint32_t valid = (vq >> (4 * (fetched - 1 - u))) & 15u;
        f32x4 vexp = {0.0f, 0.0f, 0.0f, 0.0f};
        if constexpr (kConv) vexp = *reinterpret_cast<const f32x4*>(lds.vexp[u & 1]);
        if (active) process(slot, valid, vexp);
        const bool ends = cc.t + 1 == cc.tiles || u + 1 == units;
        if (ends && active) end_item(cc.set, cc.g, cc.rb, seg_t0, cc.t + 1);
        if (u + 1 < units) {
            advance(cc);
            if (ends) seg_t0 = cc.t;
        }
    };
    fetch();
    if constexpr (kGguf) {
        // Half the waves dequantize tile u + 1, and have tile u + 2 in flight, while the others
        // use tile u: one after the other in each wave, the two took 2.8 us a tile, with
        // few rows and with many (head_dim 128)
        if (w >= CW) {
            load(0);
            stage(0);
            if (loaded < units) load(0);
            meet();
            for (int u = 0; u < units; ++u) {
                if (u + 1 < units) stage((u + 1) & 1);
                if (loaded < units) load(0);
                meet();
            }
        } else {
            fetch();
            begin_item(first);
            meet();
            for (int u = 0; u < units; ++u) {
                if (u > 0 && cc.t == 0) begin_item(desc_of(cc.set));
                use(u, u & 1);
                fetch();
                meet();
            }
        }
    } else {
        // Tile u in slot u % NS, the next NS - 1 in flight while it runs.  The barrier makes tile
        // u visible and shows slot (u - 1) % NS free, which then receives tile u + NS - 1.
        load(0);
        if (NS == 3 && loaded < units) load(1);
        begin_item(first);  // (its reads overlap the first tile's)
        if constexpr (kConv) {
            landed(0);
            convert(0, 0);
        }
        uint32_t slot = 0, fill = NS - 1;
        for (int u = 0; u < units; ++u) {
            if constexpr (!kConv) landed(u);
            meet();
            if (u > 0 && cc.t == 0) begin_item(desc_of(cc.set));
            if (loaded < units) load(fill);
            use(u, slot);
            slot = slot == NS - 1 ? 0 : slot + 1;
            fill = fill == NS - 1 ? 0 : fill + 1;
            if constexpr (kConv) {
                if (u + 1 < units) {
                    landed(u + 1);
                    convert(slot, (u + 1) & 1);
                }
            }
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (bad_seen) rerun(start, units);
}

template <int D, int SRC, bool QBF>
int launch_tile(const TileParams& p, unsigned grid, hipStream_t s) {
    hipLaunchKernelGGL((shared_tile_kernel<D, SRC, QBF>), dim3(grid), dim3(64 * kTileWaves), 0, s, p);
    VMC_LAUNCH_CHECK();
    return VMC_OK;
}

template <int D>
int dispatch_tile(const TileParams& p, int src, bool qbf, unsigned grid, hipStream_t s) {
    switch (src) {
        case TS_LOCAL:
            return qbf ? launch_tile<D, TS_LOCAL, true>(p, grid, s) : launch_tile<D, TS_LOCAL, false>(p, grid, s);
        case TS_PAGED:
            return qbf ? launch_tile<D, TS_PAGED, true>(p, grid, s) : launch_tile<D, TS_PAGED, false>(p, grid, s);
        case TS_Q8: return qbf ? launch_tile<D, TS_Q8, true>(p, grid, s) : launch_tile<D, TS_Q8, false>(p, grid, s);
        case TS_Q4: return qbf ? launch_tile<D, TS_Q4, true>(p, grid, s) : launch_tile<D, TS_Q4, false>(p, grid, s);
        default: return VMC_EINVAL;
    }
}

}  // namespace
}  // namespace vmc
