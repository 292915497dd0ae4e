// The 16-bit matrix-core backward over packed sequences: the kernels of
// sdpa_bwd_mfma.hip instantiated in a translation unit of their own.  (Their
// phase-timer instrumentation covers the other instances only.)
#undef MFX_PHASE_TIMERS
#define MFX_PACKED 1
#include "sdpa_bwd_mfma.hip"
