#define CACHE4_DP 160
#include "cache4_attention.inc"
