// attention_token.cuh -- the form of ww_cross_attention for a few query rows
// per key head (attention_token.cu).
#pragma once

#include "attention.cuh"

namespace ww {

// Whether a call takes this form: at most 32 rows (query heads of a key head x
// tokens) share each key, and sharing or few items make it pay (attention_token.cu).
bool token_form(const ww_attention_t& p, int sms) noexcept;

// CTAs that share the keys of one batch item and key head.
int token_splits(const ww_attention_t& p, int sms) noexcept;

// splits > 1: writes part_o [B * Hk][splits][rows][D] (each normalised) and
// part_lse [B * Hk][splits][rows] (log2), rows = (shared head, token), instead of
// out and lse.
int attention_token_launch(const ww_attention_t& p, int splits, float* part_o, float* part_lse,
                           cudaStream_t stream) noexcept;

}  // namespace ww
