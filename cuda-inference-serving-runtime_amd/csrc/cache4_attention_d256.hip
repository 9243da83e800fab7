#define CACHE4_DP 256
#include "cache4_attention.inc"
