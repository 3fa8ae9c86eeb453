// ffn_f32.hip - the gated feed-forward block's kernels for f32 elements.
#include "ffn_kernel.h"

template int carl::launchProduct<float>(int, const carl::ProductArgs&, hipStream_t);
template int carl::launchThin<float>(bool, const carl::ThinArgs&, hipStream_t);
template int carl::launchOuter<float>(const carl::OuterArgs&, int, hipStream_t);
template int carl::launchPack<float>(const carl::PackArgs&, hipStream_t);
template int carl::launchSum<float>(const carl::SumArgs&, hipStream_t);
