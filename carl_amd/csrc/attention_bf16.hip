// attention_bf16.hip - the chunked linear attention kernel for bf16 rows.
#include "attention_kernel.h"

template int carl::launchAttentionOf<carl::bf16>(const carl::Pass&, int, int, bool, hipStream_t);
