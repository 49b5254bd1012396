// shared_attn.hip -- decode over a shared prefix and cross attention: the C ABI's
// entry points, and the one-wave-per-row kernel that takes every shape.
//
//   o = sum_p w_p v_p / sum_p w_p,  w_p = exp(scale q.k_p - m)
// over the row's keys p: for a decode row of length L in a group that shares S
// tokens, positions 0 .. min(L, S) - 1 through the table row of the group's
// first row and S .. L - 1 through its own; for a row of a decoder, the states
// of its sequence.  fp32 throughout (generic_row.hpp), rounded once.
#include "generic_row.hpp"
#include "shared_attn.hpp"
#include "shared_plan.hpp"

namespace vmc {
namespace {

constexpr int kRowWaves = 4;  // query heads per workgroup

// the set that holds row r: starts is non-decreasing; -1 if none does
__device__ __forceinline__ int set_of_row(const SharedArgs& a, int r, int lane) {
    for (int s0 = 0; s0 < a.nsets; s0 += 64) {
        const int s = s0 + lane;
        const uint64_t hit = __ballot(s < a.nsets && a.starts[min(s, a.nsets - 1)] <= r &&
                                      r < a.starts[min(s, a.nsets - 1) + 1]);
        if (hit) return s0 + (int)__builtin_ctzll(hit);
    }
    return -1;
}

template <int D, int SRC, bool BF>
__global__ void __launch_bounds__(64 * kRowWaves) shared_row_kernel(SharedArgs a) {
    constexpr int NPL = D / 64;
    __shared__ float qsm[kRowWaves][D];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int row = blockIdx.x, hq = blockIdx.y * kRowWaves + w;
    if (hq >= a.Hq) return;
    const int g = hq / (a.Hq / a.Hkv);
    uint16_t* op = a.out + ((int64_t)row * a.Hq + hq) * D;
    const int set = __builtin_amdgcn_readfirstlane(set_of_row(a, row, lane));

    // n keys; paged: the first `common` of them through table row `first`
    int n = 0, common = 0, first = row, base = 0;
    if constexpr (SRC == GEN_LOCAL) {
        if (set < 0) return;
        base = max(a.key_starts[set], 0);
        const int64_t end = min((int64_t)a.key_starts[set] + a.set_lens[set], (int64_t)a.num_keys);
        n = (int)max(end - base, (int64_t)0);
    } else {
        n = (int)min((int64_t)a.seq_lens[row], a.max_blocks * a.bs);
        if (set >= 0) {
            common = max(a.set_lens[set], 0);
            first = max(a.starts[set], 0);
        }
    }
    if (n <= 0) {
#pragma unroll
        for (int i = 0; i < NPL; ++i) op[lane + 64 * i] = 0;
        return;
    }
    float* qs = qsm[w];
    const uint16_t* qp = a.q + row * a.q_ts + hq * a.q_hs;
#pragma unroll
    for (int i = 0; i < NPL; ++i) qs[lane + 64 * i] = half_to_f32<BF>(qp[lane + 64 * i]);
    wave_sync();
    auto key_at = [&](int k, const uint8_t*& ke, const uint8_t*& ve) __attribute__((always_inline)) {
        if constexpr (SRC == GEN_LOCAL) {
            ke = reinterpret_cast<const uint8_t*>(a.k + ((int64_t)base + k) * a.k_ts + g * a.k_hs);
            ve = reinterpret_cast<const uint8_t*>(a.v + ((int64_t)base + k) * a.v_ts + g * a.v_hs);
            return true;
        } else {
            const int32_t pg = a.bt[(int64_t)(k < common ? first : row) * a.max_blocks + k / a.bs];
            const int64_t r = k % a.bs;
            const int64_t idx = a.hnd ? ((int64_t)pg * a.Hkv + g) * a.bs + r : ((int64_t)pg * a.bs + r) * a.Hkv + g;
            ke = a.kp + idx * a.entry;
            ve = a.vp + idx * a.entry;
            return pg >= 0;
        }
    };
    GenArgs ga = {};
    ga.scale = a.scale;
    const TQTables none = {};
    float m, l, acc[NPL];
    gen_row<D, SRC, 0, 0, BF>(ga, none, qs, lane, 0, n, key_at, m, l, acc);
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int i = 0; i < NPL; ++i) op[lane + 64 * i] = f32_to_half<BF>(acc[i] * inv);
}

template <int D, bool BF>
int launch_rows(const SharedArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)a.rows, (unsigned)((a.Hq + kRowWaves - 1) / kRowWaves)), block(64 * kRowWaves);
    switch (a.src) {
        case GEN_F16: hipLaunchKernelGGL((shared_row_kernel<D, GEN_F16, BF>), grid, block, 0, s, a); break;
        case GEN_BF16: hipLaunchKernelGGL((shared_row_kernel<D, GEN_BF16, BF>), grid, block, 0, s, a); break;
        case GEN_Q8: hipLaunchKernelGGL((shared_row_kernel<D, GEN_Q8, BF>), grid, block, 0, s, a); break;
        case GEN_Q4: hipLaunchKernelGGL((shared_row_kernel<D, GEN_Q4, BF>), grid, block, 0, s, a); break;
        case GEN_LOCAL: hipLaunchKernelGGL((shared_row_kernel<D, GEN_LOCAL, BF>), grid, block, 0, s, a); break;
        default: return VMC_EINVAL;
    }
    VMC_LAUNCH_CHECK();
    return VMC_OK;
}

int shared_rows(const SharedArgs& a, hipStream_t s) {
    switch (a.D) {
        case 64: return a.q_bf16 ? launch_rows<64, true>(a, s) : launch_rows<64, false>(a, s);
        case 128: return a.q_bf16 ? launch_rows<128, true>(a, s) : launch_rows<128, false>(a, s);
        default: return a.q_bf16 ? launch_rows<256, true>(a, s) : launch_rows<256, false>(a, s);
    }
}

bool heads_valid(int num_heads, int num_kv_heads, int head_dim) {
    return num_heads > 0 && num_kv_heads > 0 && num_heads % num_kv_heads == 0 && num_heads <= 65535 * kRowWaves &&
           (head_dim == 64 || head_dim == 128 || head_dim == 256);
}

}  // namespace
}  // namespace vmc

using namespace vmc;

extern "C" size_t vmc_shared_prefix_workspace_size(int batch_size, int num_heads, int num_kv_heads, int head_dim,
                                                   int num_groups) {
    if (batch_size <= 0 || num_groups < 0 || !heads_valid(num_heads, num_kv_heads, head_dim)) return 0;
    return shared_tiles_workspace(true, batch_size, num_groups, num_heads, num_kv_heads, head_dim);
}

extern "C" int vmc_paged_attention_shared_prefix(void* out, const void* query, const void* key_cache,
                                                 const void* value_cache, const int32_t* block_tables,
                                                 const int32_t* seq_lens, const int32_t* group_starts,
                                                 const int32_t* shared_lens, int batch_size, int num_groups,
                                                 int num_heads, int num_kv_heads, int head_dim, int block_size,
                                                 int max_num_blocks_per_req, float scale, int q_dtype, int kv_format,
                                                 int layout, void* workspace, size_t workspace_bytes,
                                                 vmc_stream_t stream) {
    if (batch_size < 0 || num_groups < 0 || !heads_valid(num_heads, num_kv_heads, head_dim)) return VMC_EINVAL;
    if (block_size <= 0 || max_num_blocks_per_req < 0 || (int64_t)max_num_blocks_per_req * block_size > 0x7fffffff)
        return VMC_EINVAL;
    if (q_dtype != VMC_DTYPE_F16 && q_dtype != VMC_DTYPE_BF16) return VMC_EINVAL;
    if (layout != VMC_LAYOUT_NHD && layout != VMC_LAYOUT_HND) return VMC_EINVAL;
    const int64_t entry = vmc_kv_entry_bytes(kv_format, head_dim);
    if (entry < 0) return VMC_EINVAL;
    if (batch_size == 0) return VMC_OK;
    if ((int64_t)batch_size * num_heads >= 1 << 24) return VMC_EINVAL;  // 2^32 work-items of 256 a row and head
    if (!out || !query || !key_cache || !value_cache || !block_tables || !seq_lens) return VMC_EINVAL;
    if (num_groups > 0 && (!group_starts || !shared_lens)) return VMC_EINVAL;
    // entries are read as 32-bit words (f16 / bf16) or 16-bit ones (GGUF)
    const uintptr_t pools = (uintptr_t)key_cache | (uintptr_t)value_cache;
    if ((pools & (kv_format == VMC_KV_F16 || kv_format == VMC_KV_BF16 ? 3 : 1)) != 0 ||
        (((uintptr_t)out | (uintptr_t)query) & 1) != 0)
        return VMC_EINVAL;
    if (workspace_bytes < vmc_shared_prefix_workspace_size(batch_size, num_heads, num_kv_heads, head_dim, num_groups))
        return VMC_ENOMEM;
    if (!workspace || ((uintptr_t)workspace & 15) != 0) return VMC_EINVAL;
    SharedArgs a = {};
    a.out = reinterpret_cast<uint16_t*>(out);
    a.q = reinterpret_cast<const uint16_t*>(query);
    a.q_ts = (int64_t)num_heads * head_dim;
    a.q_hs = head_dim;
    a.q_bf16 = q_dtype == VMC_DTYPE_BF16;
    a.src = kv_format == VMC_KV_F16 ? GEN_F16 : kv_format == VMC_KV_BF16 ? GEN_BF16 : kv_format == VMC_KV_Q8_0 ? GEN_Q8 : GEN_Q4;
    a.rows = batch_size;
    a.Hq = num_heads;
    a.Hkv = num_kv_heads;
    a.D = head_dim;
    a.scale = scale;
    a.starts = group_starts;
    a.set_lens = shared_lens;
    a.nsets = num_groups;
    a.kp = reinterpret_cast<const uint8_t*>(key_cache);
    a.vp = reinterpret_cast<const uint8_t*>(value_cache);
    a.entry = entry;
    a.bs = block_size;
    a.max_blocks = max_num_blocks_per_req;
    a.hnd = layout == VMC_LAYOUT_HND;
    a.bt = block_tables;
    a.seq_lens = seq_lens;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    return shared_tiles_take(a) ? shared_tiles(a, workspace, s) : shared_rows(a, s);
}

extern "C" size_t vmc_cross_attention_workspace_size(int num_tokens, int num_seqs, int num_heads, int num_kv_heads,
                                                     int head_dim) {
    if (num_tokens <= 0 || num_seqs <= 0 || !heads_valid(num_heads, num_kv_heads, head_dim)) return 0;
    return shared_tiles_workspace(false, num_tokens, num_seqs, num_heads, num_kv_heads, head_dim);
}

extern "C" int vmc_cross_attention(void* out, const void* query, const void* key, const void* value,
                                   const int32_t* query_starts, const int32_t* key_starts, const int32_t* key_lens,
                                   int num_tokens, int num_keys, int num_seqs, int num_heads, int num_kv_heads,
                                   int head_dim, int64_t query_token_stride, int64_t query_head_stride,
                                   int64_t key_token_stride, int64_t key_head_stride, int64_t value_token_stride,
                                   int64_t value_head_stride, float scale, int dtype, void* workspace,
                                   size_t workspace_bytes, vmc_stream_t stream) {
    if (num_tokens < 0 || num_keys < 0 || num_seqs < 0 || !heads_valid(num_heads, num_kv_heads, head_dim))
        return VMC_EINVAL;
    if (dtype != VMC_DTYPE_F16 && dtype != VMC_DTYPE_BF16) return VMC_EINVAL;
    // a stride of fewer values than a head has would overlap rows; even, as rows are read by 32-bit words
    for (int64_t st : {query_token_stride, query_head_stride, key_token_stride, key_head_stride, value_token_stride,
                       value_head_stride})
        if (st < head_dim || st % 2 != 0 || st > (int64_t)1 << 40) return VMC_EINVAL;
    if (num_tokens == 0 || num_seqs == 0) return VMC_OK;
    if (num_tokens >= 1 << 24 || (int64_t)num_tokens * num_heads > 0x7fffffff) return VMC_EINVAL;
    if (!out || !query || !query_starts || !key_starts || !key_lens) return VMC_EINVAL;
    if (num_keys > 0 && (!key || !value)) return VMC_EINVAL;
    if ((((uintptr_t)out | (uintptr_t)query) & 1) != 0 || (((uintptr_t)key | (uintptr_t)value) & 3) != 0)
        return VMC_EINVAL;
    if (workspace_bytes < vmc_cross_attention_workspace_size(num_tokens, num_seqs, num_heads, num_kv_heads, head_dim))
        return VMC_ENOMEM;
    if (!workspace || ((uintptr_t)workspace & 15) != 0) return VMC_EINVAL;
    SharedArgs a = {};
    a.out = reinterpret_cast<uint16_t*>(out);
    a.q = reinterpret_cast<const uint16_t*>(query);
    a.q_ts = query_token_stride;
    a.q_hs = query_head_stride;
    a.q_bf16 = dtype == VMC_DTYPE_BF16;
    a.src = GEN_LOCAL;
    a.rows = num_tokens;
    a.Hq = num_heads;
    a.Hkv = num_kv_heads;
    a.D = head_dim;
    a.scale = scale;
    a.starts = query_starts;
    a.set_lens = key_lens;
    a.nsets = num_seqs;
    a.k = reinterpret_cast<const uint16_t*>(key);
    a.v = reinterpret_cast<const uint16_t*>(value);
    a.k_ts = key_token_stride;
    a.k_hs = key_head_stride;
    a.v_ts = value_token_stride;
    a.v_hs = value_head_stride;
    a.key_starts = key_starts;
    a.num_keys = num_keys;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    return shared_tiles_take(a) ? shared_tiles(a, workspace, s) : shared_rows(a, s);
}
