// cm_token_f16.hip -- the kernels of cm_token.hip for f16 logits (a translation unit per type: they compile side by side)
#include "cm_token_rows.h"
int tok_launch_f16(TokArgs a, int mode, bool en, void* scratch, hipStream_t s) { return tok_launch_type<TokF16>(a, mode, en, scratch, s); }
