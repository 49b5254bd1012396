// rope_append.hip -- rotation of Q and K and append of K and V to the paged cache,
// in one pass over the fused QKV projection's rows.
//
//   a' = a cos - b sin, b' = b cos + a sin over the first rotary_dim values of a
// head, pairs (i, i + rotary_dim / 2) or (2i, 2i + 1); in fp32 from fp32 tables,
// rounded once to the element type; the other values pass.
//
// What bounds it: HBM for a prefill step, the launch and its dependent reads
// (position -> table row) for a decode step.  A head's row is D / 8 lanes of 16
// bytes; the lanes of a row exchange the pairs' other halves, so each value is
// read and written once; the table rows come from the L2.  Measured: 65 us for 16384
// tokens of 16 + 2 heads of 256 with their V (0.34 GB in and out, 5.2 TB/s, what a
// copy reaches), 7.4 us for 5003 tokens of 14 + 2 heads of 64, 3.4 us for 32
// tokens.  Several heads a lane, sharing a table row, would save reads
// that the L2 has anyway.
#include "row_codec.hpp"

namespace vmc {
namespace {

struct RopeParams {
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    int64_t q_ts, k_ts, v_ts;  // values between tokens
    uint16_t* q_out;           // [T][Hq][D], or null
    uint16_t* k_out;           // [T][Hkv][D], or null
    const float* cs;           // [max_pos][rot]
    const int64_t* pos;
    int64_t max_pos;
    uint8_t* kc;  // null: no append
    uint8_t* vc;
    const int64_t* slots;
    int T, Hq, Hkv, rot;
    int64_t bs, E, stride;
    int hnd;
};

constexpr int kNoPages = -1;

// Rows of a token: Hkv K rows (with their V rows), then Hq Q rows.  FMT: page format,
// or kNoPages.
template <int D, bool BF, int FMT, bool NEOX>
__global__ void __launch_bounds__(256) rope_append_kernel(RopeParams p) {
    constexpr int LPR = D / 8;      // lanes of a row
    constexpr int RPW = 256 / LPR;  // rows of a workgroup
    const int j = threadIdx.x % LPR;
    const uint32_t per_tok = (uint32_t)(p.Hkv + p.Hq);
    const uint32_t item = blockIdx.x * RPW + threadIdx.x / LPR;
    const int64_t t_raw = item / per_tok;
    // lanes past the end follow the last token without writing (they take part
    // in the exchanges of their wave)
    const int64_t t = min(t_raw, (int64_t)p.T - 1);
    const int row = (int)(item % per_tok);
    const bool is_k = row < p.Hkv;
    const int h = is_k ? row : row - p.Hkv;

    const int64_t pos = p.pos[t];
    const bool live = t_raw < p.T && pos >= 0 && pos < p.max_pos;
    const uint16_t* src = (is_k ? p.k + t * p.k_ts : p.q + t * p.q_ts) + (int64_t)h * D + 8 * j;
    const u32x4 xr = *reinterpret_cast<const u32x4*>(src);
    u32x4 vr = {0u, 0u, 0u, 0u};
    int64_t slot = -1;
    if constexpr (FMT != kNoPages) {
        if (is_k) {
            vr = *reinterpret_cast<const u32x4*>(p.v + t * p.v_ts + (int64_t)h * D + 8 * j);
            if (live) slot = p.slots[t];
        }
    }
    // ---- this lane's rotation: 8 values of cos and sin (NEOX: of the chunk's
    // pairs; else 4 pairs, each for two values)
    const int half = p.rot >> 1, hc = half >> 3;  // chunks of a half (NEOX)
    const bool turns = 8 * j < p.rot;
    const bool lower = NEOX && j >= hc;  // the chunk holds the pairs' second values
    const int mate = NEOX ? (turns ? (lower ? j - hc : j + hc) : j) : j;
    constexpr int NC = NEOX ? 8 : 4;
    float c[NC], s[NC];
    {
        const float* cs = p.cs + (live ? pos : 0) * p.rot;
        const int at = turns ? (NEOX ? 8 * (lower ? j - hc : j) : 4 * j) : 0;
#pragma unroll
        for (int e = 0; e < NC; e += 4) {
            const f32x4 cv = *reinterpret_cast<const f32x4*>(cs + at + e);
            const f32x4 sv = *reinterpret_cast<const f32x4*>(cs + half + at + e);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                c[e + i] = cv[i];
                s[e + i] = sv[i];
            }
        }
    }
    const int mate_lane = (int)(threadIdx.x & 63) - j + mate;
    float x[8], y[8];
    unpack8<BF>(xr, x);
    if constexpr (NEOX) {
        u32x4 ow;
#pragma unroll
        for (int e = 0; e < 4; ++e) ow[e] = (uint32_t)__shfl((int)xr[e], mate_lane, kWave);
        float o[8];
        unpack8<BF>(ow, o);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float t0 = x[e] * c[e], t1 = o[e] * s[e];
            y[e] = lower ? t0 + t1 : t0 - t1;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = x[2 * i], b = x[2 * i + 1];
            y[2 * i] = a * c[i] - b * s[i];
            y[2 * i + 1] = b * c[i] + a * s[i];
        }
    }
    const u32x4 turned = pack8<BF>(y);
    const u32x4 yw = turns ? turned : xr;  // values that do not turn keep their bits
    const int64_t at = (t * (is_k ? p.Hkv : p.Hq) + h) * D + 8 * j;
    uint16_t* dst = is_k ? p.k_out : p.q_out;
    if (live && dst) *reinterpret_cast<u32x4*>(dst + at) = yw;
    if constexpr (FMT != kNoPages) {
        if (!is_k) return;
        const bool wr = slot >= 0;
        const int64_t eo = kv_entry_offset(wr ? slot : 0, h, p.bs, p.Hkv, p.E, p.stride, p.hnd != 0);
        if constexpr (FMT == VMC_KV_F16 || FMT == VMC_KV_BF16) {
            constexpr bool DB = FMT == VMC_KV_BF16;
            u32x4 kw = yw, vw = vr;
            if constexpr (DB != BF) {
                float f[8];
                unpack8<BF>(yw, f);
                kw = pack8<DB>(f);
                unpack8<BF>(vr, f);
                vw = pack8<DB>(f);
            }
            if (wr) {
                *reinterpret_cast<u32x4*>(p.kc + eo + 16 * j) = kw;
                *reinterpret_cast<u32x4*>(p.vc + eo + 16 * j) = vw;
            }
        } else {
            float f[8];
            unpack8<BF>(yw, f);
            gguf_block4<FMT>(f, j, p.kc + eo, wr);
            unpack8<BF>(vr, f);
            gguf_block4<FMT>(f, j, p.vc + eo, wr);
        }
    }
}

template <int D, bool BF, int FMT, bool NEOX>
int launch_rope(const RopeParams& p, hipStream_t s) {
    const int64_t items = (int64_t)p.T * ((int64_t)p.Hkv + p.Hq);
    if (items >= ((int64_t)1 << 32) / (D / 8) - 256) return VMC_EINVAL;  // a launch has 2^32 work-items at most
    const int64_t grid = (items + 256 / (D / 8) - 1) / (256 / (D / 8));
    hipLaunchKernelGGL((rope_append_kernel<D, BF, FMT, NEOX>), dim3((unsigned)grid), dim3(256), 0, s, p);
    VMC_LAUNCH_CHECK();
    return VMC_OK;
}

template <int D, bool BF, int FMT>
int dispatch_pairs(const RopeParams& p, bool neox, hipStream_t s) {
    return neox ? launch_rope<D, BF, FMT, true>(p, s) : launch_rope<D, BF, FMT, false>(p, s);
}

template <int D, bool BF>
int dispatch_format(const RopeParams& p, int fmt, bool neox, hipStream_t s) {
    switch (fmt) {
        case kNoPages: return dispatch_pairs<D, BF, kNoPages>(p, neox, s);
        case VMC_KV_F16: return dispatch_pairs<D, BF, VMC_KV_F16>(p, neox, s);
        case VMC_KV_BF16: return dispatch_pairs<D, BF, VMC_KV_BF16>(p, neox, s);
        case VMC_KV_Q8_0: return dispatch_pairs<D, BF, VMC_KV_Q8_0>(p, neox, s);
        case VMC_KV_Q4_0: return dispatch_pairs<D, BF, VMC_KV_Q4_0>(p, neox, s);
        default: return VMC_EINVAL;
    }
}

template <int D>
int dispatch_type(const RopeParams& p, int fmt, bool neox, bool bf, hipStream_t s) {
    return bf ? dispatch_format<D, true>(p, fmt, neox, s) : dispatch_format<D, false>(p, fmt, neox, s);
}

}  // namespace
}  // namespace vmc

using namespace vmc;

extern "C" int vmc_rope_and_cache(void* query_out, void* key_out, const void* query, const void* key,
                                  const void* value, const float* cos_sin, const int64_t* position_ids,
                                  void* key_cache, void* value_cache, const int64_t* slot_mapping, int num_tokens,
                                  int num_heads, int num_kv_heads, int head_dim, int rotary_dim, int64_t max_position,
                                  int64_t query_token_stride, int64_t key_token_stride, int64_t value_token_stride,
                                  int is_neox, int64_t block_size, int64_t cache_stride, int kv_format, int layout,
                                  int dtype, vmc_stream_t stream) {
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return VMC_EINVAL;
    if (rotary_dim < 16 || rotary_dim > head_dim || rotary_dim % 16 != 0) return VMC_EINVAL;
    if (num_tokens < 0 || num_heads <= 0 || num_kv_heads <= 0 || max_position <= 0) return VMC_EINVAL;
    if (dtype != VMC_DTYPE_F16 && dtype != VMC_DTYPE_BF16) return VMC_EINVAL;
    // rows are read and written 16 bytes at a time
    if (query_token_stride < (int64_t)num_heads * head_dim || key_token_stride < (int64_t)num_kv_heads * head_dim ||
        query_token_stride % 8 != 0 || key_token_stride % 8 != 0)
        return VMC_EINVAL;
    if (num_tokens == 0) return VMC_OK;
    if (!query_out || !query || !key || !cos_sin || !position_ids || (!key_out && !key_cache)) return VMC_EINVAL;
    if ((((uintptr_t)query_out | (uintptr_t)key_out | (uintptr_t)query | (uintptr_t)key | (uintptr_t)cos_sin) & 15) != 0)
        return VMC_EINVAL;
    RopeParams p = {};
    p.q = reinterpret_cast<const uint16_t*>(query);
    p.k = reinterpret_cast<const uint16_t*>(key);
    p.q_ts = query_token_stride;
    p.k_ts = key_token_stride;
    p.q_out = reinterpret_cast<uint16_t*>(query_out);
    p.k_out = reinterpret_cast<uint16_t*>(key_out);
    p.cs = cos_sin;
    p.pos = position_ids;
    p.max_pos = max_position;
    p.T = num_tokens;
    p.Hq = num_heads;
    p.Hkv = num_kv_heads;
    p.rot = rotary_dim;
    int fmt = kNoPages;
    if (key_cache) {
        const int64_t E = vmc_kv_entry_bytes(kv_format, head_dim);
        if (E < 0 || (layout != VMC_LAYOUT_NHD && layout != VMC_LAYOUT_HND)) return VMC_EINVAL;
        if (!value || !value_cache || !slot_mapping || block_size <= 0) return VMC_EINVAL;
        if (value_token_stride < (int64_t)num_kv_heads * head_dim || value_token_stride % 8 != 0 ||
            ((uintptr_t)value & 15) != 0)
            return VMC_EINVAL;
        p.stride = cache_stride > 0 ? cache_stride : block_size * num_kv_heads * E;
        if (p.stride < block_size * num_kv_heads * E) return VMC_EINVAL;
        // f16 / bf16 entries take 16-byte stores, GGUF ones 16-bit stores
        const int64_t a = kv_format == VMC_KV_F16 || kv_format == VMC_KV_BF16 ? 16 : 2;
        if (p.stride % a != 0 || ((uintptr_t)key_cache | (uintptr_t)value_cache) % (uintptr_t)a != 0) return VMC_EINVAL;
        p.v = reinterpret_cast<const uint16_t*>(value);
        p.v_ts = value_token_stride;
        p.kc = reinterpret_cast<uint8_t*>(key_cache);
        p.vc = reinterpret_cast<uint8_t*>(value_cache);
        p.slots = slot_mapping;
        p.bs = block_size;
        p.E = E;
        p.hnd = layout == VMC_LAYOUT_HND;
        fmt = kv_format;
    }
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const bool neox = is_neox != 0, bf = dtype == VMC_DTYPE_BF16;
    return head_dim == 64    ? dispatch_type<64>(p, fmt, neox, bf, s)
           : head_dim == 128 ? dispatch_type<128>(p, fmt, neox, bf, s)
                             : dispatch_type<256>(p, fmt, neox, bf, s);
}
