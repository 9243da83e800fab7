#define CACHE4_DP 192
#include "cache4_attention.inc"
