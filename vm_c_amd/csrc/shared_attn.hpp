// shared_attn.hpp -- attention of several rows over one set of keys, without a
// causal mask: sets are groups of decode rows with a common prefix in the paged
// cache (plus each row's own pages), or sequences of decoder rows over an
// encoder's states.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "generic_attn.hpp"
#include "vmc_attn.h"

namespace vmc {

struct SharedArgs {
    uint16_t* out;  // [rows][Hq][D]
    const uint16_t* q;
    int64_t q_ts, q_hs;  // values between rows, between heads
    int q_bf16;          // q / out type (GEN_LOCAL: also K / V)
    int src;             // GenSrc
    int rows, Hq, Hkv, D;
    float scale;
    // set s: rows starts[s] .. starts[s + 1] - 1 over set_lens[s] common keys
    const int32_t* starts;
    const int32_t* set_lens;
    int nsets;
    // pages: the common keys through the table row of the set's first row, the
    // others up to seq_lens[row] through the row's own; rows of no set have
    // their own keys alone
    const uint8_t* kp;
    const uint8_t* vp;
    int64_t entry, bs, max_blocks;
    int hnd;
    const int32_t* bt;
    const int32_t* seq_lens;
    // contiguous keys (GEN_LOCAL): key i of set s is row key_starts[s] + i of
    // num_keys; rows of no set are left alone
    const uint16_t* k;
    const uint16_t* v;
    int64_t k_ts, k_hs, v_ts, v_hs;  // values between keys, between heads
    const int32_t* key_starts;
    int num_keys;
};

}  // namespace vmc
