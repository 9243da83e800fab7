#define CACHE4_DP 128
#include "cache4_attention.inc"
