#define CACHE4_DP 64
#include "cache4_attention.inc"
