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

// ww_cross_attention.  `powers`, not nullptr only for fp16 calls that are not of the token form: keys and values come divided by
// powers of two, which scores and results take back: what those of each (batch item, key head) are to be multiplied by,
// [B][Hk] {keys, values}.  (attention_forward.cu)
int cross_attention(const ww_attention_t& p, const float2* powers, void* stream) noexcept;

// Joins such parts into out and lse; launched behind the kernel that writes them
// (attention_forward.cu).
int attention_join_launch(const ww_attention_t& p, int items, int splits, int rows, const float* part_o, const float* part_lse,
                          const char* name, cudaStream_t stream) noexcept;

}  // namespace ww
