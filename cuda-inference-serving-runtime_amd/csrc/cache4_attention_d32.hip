#define CACHE4_DP 32
#include "cache4_attention.inc"
