// cm_token_f32.hip -- the kernels of cm_token.hip for f32 logits (a translation unit per type: they compile side by side)
#include "cm_token_rows.h"
int tok_launch_f32(TokArgs a, int mode, bool en, void* scratch, hipStream_t s) { return tok_launch_type<TokF32>(a, mode, en, scratch, s); }
