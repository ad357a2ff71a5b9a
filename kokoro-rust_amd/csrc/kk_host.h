// kk_host.h -- host-only rules of the library: the ragged layout tables, the duration rule and the
// checks of an ids-level item.  No HIP in these files (kk_host.cpp), so the same source also builds
// with a plain C++ compiler under AddressSanitizer / UndefinedBehaviorSanitizer for the CPU tests.
#pragma once
#include <cstdint>
#include <string>

#include "kokoro_hip.h"

namespace kk {

constexpr int kGapN = 2;  // GAP_N (src/gpu_batch.rs:27): gap frames after each item
constexpr int kGapT = 2;  // GAP_T (src/gpu_batch.rs:29): gap token rows after each item

// The refusal of one ids-level item (src/gpu_batch.rs:182-187: null inputs, input_ids length
// outside [2, 512], an id outside the vocabulary, speed not positive and finite, an unknown noise
// kind), or "" for an item the forward accepts.  The fixed noise's length is checked against the
// predicted frames later.
std::string ids_item_error(const kk_item& it, int b);

// The refusals of the operators over an 8-bit cache, or "": what the host can see of their arguments (sizes, types, null
// pointers, alignment, and sizes that a launch could not hold).
std::string norm_rope_error(const kk_norm_rope* a);
std::string kv_batch_error(const kk_kv_cache* c, const kk_kv_batch* b);
std::string kv_rows_error(const kk_kv_rows* r);
std::string kv_attention_error(const kk_kv_cache* c, const kk_kv_batch* b, const kk_kv_attention_args* a);

// The same of the products of ragged rows.
std::string expert_route_error(const kk_expert_route_args* a);
std::string expert_product_error(const kk_expert_product_args* a);
std::string expert_join_error(const kk_expert_join_args* a);
std::string adapter_product_error(const kk_adapter_product_args* a);

}  // namespace kk
