// The pipelined flash kernel over packed sequences: the kernel of
// sdpa_flash_bf16_pipe.hip instantiated in a translation unit of its own.
// (Its phase-timer instrumentation covers the other instances only.)
#undef MFX_PHASE_TIMERS
#define MFX_PACKED 1
#include "sdpa_flash_bf16_pipe.hip"
