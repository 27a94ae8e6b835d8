// The instances of paged_decode_kernel for scores that are capped, biased by distance, or seen by ranges of the tokens' own: the same source in a translation unit of its
// own (each takes a minute and a half to compile).
#define B200KV_PAGED_DECODE_SCORED
#include "paged_decode.cu"
