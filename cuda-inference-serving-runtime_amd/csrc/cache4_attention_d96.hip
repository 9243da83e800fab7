#define CACHE4_DP 96
#include "cache4_attention.inc"
