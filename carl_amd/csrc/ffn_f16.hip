// ffn_f16.hip - the gated feed-forward block's kernels for f16 elements.
#include "ffn_kernel.h"

template int carl::launchProduct<carl::f16>(int, const carl::ProductArgs&, hipStream_t);
template int carl::launchThin<carl::f16>(bool, const carl::ThinArgs&, hipStream_t);
template int carl::launchOuter<carl::f16>(const carl::OuterArgs&, int, hipStream_t);
template int carl::launchPack<carl::f16>(const carl::PackArgs&, hipStream_t);
template int carl::launchSum<carl::f16>(const carl::SumArgs&, hipStream_t);
