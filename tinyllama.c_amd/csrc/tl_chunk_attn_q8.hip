/* chunk attention and attention weight: the instances over a q8 cache */
#include "tl_chunk_attn_kernels.h"
#include "tl_chunk_launch.h"
#include "tl_chunk_weight_kernels.h"

template <int D, bool Q8>
void ck_launch_attn_t(const CkAttnParams &p, u32 wgs, hipStream_t st) {
    if (p.softcap > 0.f || p.slopes)
        hipLaunchKernelGGL((chunk_attn_kernel<D, Q8, true>), dim3(wgs), dim3(64 * CK_WAVES(D)), 0, st, p);
    else
        hipLaunchKernelGGL((chunk_attn_kernel<D, Q8, false>), dim3(wgs), dim3(64 * CK_WAVES(D)), 0, st, p);
}
template <int D, bool Q8>
void ck_launch_both_t(const CkAttnParams &p, u32 wgs, hipStream_t st) {
    if (p.softcap > 0.f || p.slopes)
        hipLaunchKernelGGL((chunk_attn_both_kernel<D, Q8, true>), dim3(wgs), dim3(256), 0, st, p);
    else
        hipLaunchKernelGGL((chunk_attn_both_kernel<D, Q8, false>), dim3(wgs), dim3(256), 0, st, p);
}
template <int D, bool Q8>
void ck_launch_wide_t(const CkAttnParams &p, u32 wgs, hipStream_t st) {
    if (p.softcap > 0.f || p.slopes)
        hipLaunchKernelGGL((chunk_attn_wide_kernel<D, Q8, true>), dim3(wgs), dim3(CkWide<D, Q8>::NT), 0, st, p);
    else
        hipLaunchKernelGGL((chunk_attn_wide_kernel<D, Q8, false>), dim3(wgs), dim3(CkWide<D, Q8>::NT), 0, st, p);
}
template <int D, bool Q8>
void ck_launch_weight_t(const CkAttnParams &p, u32 wgs, hipStream_t st) {
    if (p.softcap > 0.f || p.slopes)
        hipLaunchKernelGGL((chunk_weight_kernel<D, Q8, true>), dim3(wgs), dim3(512), 0, st, p);
    else
        hipLaunchKernelGGL((chunk_weight_kernel<D, Q8, false>), dim3(wgs), dim3(512), 0, st, p);
}
template <int D, bool Q8>
void ck_launch_weight_wide_t(const CkAttnParams &p, u32 wgs, hipStream_t st) {
    if (p.softcap > 0.f || p.slopes)
        hipLaunchKernelGGL((chunk_weight_wide_kernel<D, Q8, true>), dim3(wgs), dim3(512), 0, st, p);
    else
        hipLaunchKernelGGL((chunk_weight_wide_kernel<D, Q8, false>), dim3(wgs), dim3(512), 0, st, p);
}
template void ck_launch_attn_t<64, true>(const CkAttnParams &, u32, hipStream_t);
template void ck_launch_attn_t<128, true>(const CkAttnParams &, u32, hipStream_t);
template void ck_launch_attn_t<256, true>(const CkAttnParams &, u32, hipStream_t);
template void ck_launch_weight_t<64, true>(const CkAttnParams &, u32, hipStream_t);
template void ck_launch_weight_t<128, true>(const CkAttnParams &, u32, hipStream_t);
template void ck_launch_weight_t<256, true>(const CkAttnParams &, u32, hipStream_t);
template void ck_launch_weight_wide_t<64, true>(const CkAttnParams &, u32, hipStream_t);
template void ck_launch_both_t<64, true>(const CkAttnParams &, u32, hipStream_t);
template void ck_launch_wide_t<64, true>(const CkAttnParams &, u32, hipStream_t);
template void ck_launch_weight_wide_t<128, true>(const CkAttnParams &, u32, hipStream_t);
template void ck_launch_both_t<128, true>(const CkAttnParams &, u32, hipStream_t);
template void ck_launch_wide_t<128, true>(const CkAttnParams &, u32, hipStream_t);
template void ck_launch_weight_wide_t<256, true>(const CkAttnParams &, u32, hipStream_t);
template void ck_launch_wide_t<256, true>(const CkAttnParams &, u32, hipStream_t);
