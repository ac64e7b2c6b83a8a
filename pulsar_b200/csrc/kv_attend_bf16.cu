/* kv_attend_bf16.cu - attention over bf16 caches (pk_attend.cuh) */
#include "pk_attend.cuh"

pk_attend_fn pk_attend_bf16(int dp, int r, bool wide) { return pk_attend_pick<PULSAR_TYPE_BF16>(dp, r, wide); }
