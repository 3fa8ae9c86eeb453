// attention_f16.hip - the chunked linear attention kernel for f16 rows.
#include "attention_kernel.h"

template int carl::launchAttentionOf<carl::f16>(const carl::Pass&, int, int, bool, hipStream_t);
