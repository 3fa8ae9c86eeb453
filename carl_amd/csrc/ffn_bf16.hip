// ffn_bf16.hip - the gated feed-forward block's kernels for bf16 elements.
#include "ffn_kernel.h"

template int carl::launchProduct<carl::bf16>(int, const carl::ProductArgs&, hipStream_t);
template int carl::launchThin<carl::bf16>(bool, const carl::ThinArgs&, hipStream_t);
template int carl::launchOuter<carl::bf16>(const carl::OuterArgs&, int, hipStream_t);
template int carl::launchPack<carl::bf16>(const carl::PackArgs&, hipStream_t);
template int carl::launchSum<carl::bf16>(const carl::SumArgs&, hipStream_t);
