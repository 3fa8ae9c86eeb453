// attention_f32.hip - the chunked linear attention kernel for f32 rows.
#include "attention_kernel.h"

template int carl::launchAttentionOf<float>(const carl::Pass&, int, int, bool, hipStream_t);
