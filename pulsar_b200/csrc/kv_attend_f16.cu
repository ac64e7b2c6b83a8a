/* kv_attend_f16.cu - attention over f16 caches (pk_attend.cuh) */
#include "pk_attend.cuh"

pk_attend_fn pk_attend_f16(int dp, int r, bool wide) { return pk_attend_pick<PULSAR_TYPE_F16>(dp, r, wide); }
