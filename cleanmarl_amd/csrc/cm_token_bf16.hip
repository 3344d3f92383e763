// cm_token_bf16.hip -- the kernels of cm_token.hip for bf16 logits (a translation unit per type: they compile side by side)
#include "cm_token_rows.h"
int tok_launch_bf16(TokArgs a, int mode, bool en, void* scratch, hipStream_t s) { return tok_launch_type<TokBF16>(a, mode, en, scratch, s); }
