#define CACHE4_DP 224
#include "cache4_attention.inc"
