/* tl_chunk_launch.h — launches of the chunk kernels; their instances are
 * spread over several translation units. */
#pragma once
#include "tl_chunk.h"

void ck_launch_attn(const CkAttnParams &p, u32 head_dim, bool q8, u32 wgs, hipStream_t st);
void ck_launch_weight(const CkAttnParams &p, u32 head_dim, bool q8, u32 wgs, hipStream_t st);
template <int D, bool Q8>
void ck_launch_attn_t(const CkAttnParams &p, u32 wgs, hipStream_t st);
void ck_launch_wide(const CkAttnParams &p, u32 head_dim, bool q8, u32 wgs, hipStream_t st);
void ck_launch_merge(const CkAttnParams &p, u32 head_dim, u32 wgs, hipStream_t st);
template <int D, bool Q8>
void ck_launch_wide_t(const CkAttnParams &p, u32 wgs, hipStream_t st);
template <int D, bool Q8>
void ck_launch_weight_t(const CkAttnParams &p, u32 wgs, hipStream_t st);
void ck_launch_weight_wide(const CkAttnParams &p, u32 head_dim, bool q8, u32 wgs, hipStream_t st);
template <int D, bool Q8>
void ck_launch_weight_wide_t(const CkAttnParams &p, u32 wgs, hipStream_t st);
void ck_launch_both(const CkAttnParams &p, u32 head_dim, bool q8, u32 wgs, hipStream_t st);
template <int D, bool Q8>
void ck_launch_both_t(const CkAttnParams &p, u32 wgs, hipStream_t st);
