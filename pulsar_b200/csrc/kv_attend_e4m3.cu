/* kv_attend_e4m3.cu - attention over e4m3 caches (pk_attend.cuh) */
#include "pk_attend.cuh"

pk_attend_fn pk_attend_e4m3(int dp, int r, bool wide) { return pk_attend_pick<PULSAR_TYPE_E4M3>(dp, r, wide); }
