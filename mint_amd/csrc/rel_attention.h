// Attention with a sliding window, sinks and a learned relative position bias by buckets (include/fact_hip.h FactAttention),
// and the per-head norm of queries and keys with rotation (FactQkNorm): checks and launches.  0 = ok, negative = error with
// the reason in *why.
#pragma once
#include "../../include/fact_hip.h"
#include "common.h"

int rel_attention_check(const FactAttention& a, bool backward, const char** why);
size_t rel_attention_ws(const FactAttention& a, bool backward);  // bytes, of a checked call
int launch_rel_attention_fwd(const FactAttention& a, void* ws, hipStream_t s);
int launch_rel_attention_bwd(const FactAttention& a, void* ws, hipStream_t s);

// rows t0 .. n - 1 of every sequence of a [B * n][ld] bf16 matrix: `width` columns (a multiple of 8) cleared
int launch_zero_rows(bf16_t* x, int B, int n, int t0, int ld, int width, hipStream_t s);

int qk_norm_check(const FactQkNorm& a, bool backward, const char** why);
size_t qk_norm_ws(const FactQkNorm& a, bool backward);
int launch_qk_norm_fwd(const FactQkNorm& a, hipStream_t s);
int launch_qk_norm_bwd(const FactQkNorm& a, void* ws, hipStream_t s);

// fact_relative_buckets: -1 on bad arguments
int relative_buckets(int num_buckets, int max_distance, int bidirectional, int32_t* map);
