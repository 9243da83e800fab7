// Writing into the cache that is held in 4 bits, reading it back, and giving up the keys with the least attention weight.
//
// Write: q' = rot(q) goes to rows of its own, rot(k) and v to the pages.  A thread has 8 coordinates, four threads a block; the
// block's scale follows from its largest magnitude a alone: 2^s with a / 2^s in (3.5, 7], which is the exponent of a after
// a quarter of its leading bit has been added (normal numbers: 11.2 % off; the limits 6 and 8 give 11.5 %).  The rotary sums are rounded
// product by product, without fused steps, so that a code near a border does not depend on how a compiler joins them.
// An infinity is held as the largest number of the largest scale, a NaN as zero: what is cached is always finite.
// Bound by the bytes of the rows: 2,048 rows of 32 heads and 2 times 8 of 128 in 12 us, 3.8 TB/s; eight rows by the launch, 4 us.
#include "cache4.h"
#include <type_traits>

struct Write4Args {
    const void* qkv; const int* positions; const int* slots; const float* cos; const float* sin;
    uint8_t* pages; void* q;
    int rows, heads, kv_heads, dim, dp, rot, shift, max_pos, n_pages, interleaved;
};

// Codes of 8 coordinates and, from the four threads of a block, its scale.
__device__ __forceinline__ uint32_t cache4_codes(const float (&x)[8], int& s) {
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(x[i]));
    most = fmaxf(most, __shfl_xor(most, 1, WAVE));
    most = fmaxf(most, __shfl_xor(most, 2, WAVE));
    s = min(max((int)((__float_as_uint(most) + 0x1fffffu) >> 23) - 129, -125), 125);
    // the conversion rounds to the nearest, ties to the even code, and stops at 6; it takes a NaN for 6 and keeps the sign of a zero
    float sum = 0.f, y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) { y[i] = x[i] + 0.f; sum += y[i]; }
    if (sum != sum)
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = x[i] != x[i] ? 0.f : y[i];
    const float scale = __uint_as_float((uint32_t)(127 + s) << 23);
    uint32_t word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, y[0], y[1], scale, 0);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, y[2], y[3], scale, 1);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, y[4], y[5], scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, y[6], y[7], scale, 3);
}

// Eight coordinates from c0 on of a token's key or value, with their scale, to their places.  (The four threads of a block call it together.)
__device__ __forceinline__ void cache4_put(const Write4Args& p, int slot, int head, bool value, int c0, const float (&y)[8]) {
    int s;
    const uint32_t word = cache4_codes(y, s);
    if (slot < 0 || slot >> p.shift >= p.n_pages) return;
    const int t = slot & ((1 << p.shift) - 1);
    uint8_t* page = p.pages + ((size_t)(slot >> p.shift) * p.kv_heads + head) * cache4_record(p.dp, 1 << p.shift);
    if (c0 % 32 == 0) page[cache4_scale_at(p.dp, p.shift, t, c0 / 32, value)] = (uint8_t)(s + CACHE4_BIAS);
    if (!value) {
        *(uint32_t*)(page + cache4_key_at(p.dp, t, c0)) = word;
        return;
    }
    const int w = cache4_cut(p.dp) / 16;
    if (w == 8) {
        *(uint32_t*)(page + cache4_value_at(p.dp, p.shift, t, c0)) = word;
    } else if (w == 4) {
        for (int i = 0; i < 2; ++i) *(uint16_t*)(page + cache4_value_at(p.dp, p.shift, t, c0 + 4 * i)) = (uint16_t)(word >> (16 * i));
    } else {
        for (int i = 0; i < 4; ++i) page[cache4_value_at(p.dp, p.shift, t, c0 + 2 * i)] = (uint8_t)(word >> (8 * i));
    }
}

// Whole heads turn, in halves of whole blocks: a thread has eight coordinates of either half, the pairs that turn together.
template <typename T>
__global__ void __launch_bounds__(256)
write4_halves_kernel(Write4Args p) {
#pragma clang fp contract(off)
    const uint32_t per_head = p.dim / 16, all = p.heads + 2 * p.kv_heads, at = blockIdx.x * 256 + threadIdx.x, vector = at / per_head, row = vector / all;
    if (row >= (uint32_t)p.rows) return;                           // (whole blocks of 32 coordinates: their four threads leave together)
    const int c0 = 8 * (int)(at - vector * per_head), h = (int)(vector - row * all), half = p.dim / 2;
    const T* x = (const T*)p.qkv + (size_t)vector * p.dim;
    float a[8], b[8];
    load_run<4>(x + c0, *(float (*)[4])a); load_run<4>(x + c0 + 4, *(float (*)[4])(a + 4));
    load_run<4>(x + half + c0, *(float (*)[4])b); load_run<4>(x + half + c0 + 4, *(float (*)[4])(b + 4));
    const bool value = h >= p.heads + p.kv_heads;
    if (!value) {
        const size_t pos = (size_t)min(max(p.positions[row], 0), p.max_pos - 1) * half + c0;
        float cs[8], sn[8];
        load_run<4>(p.cos + pos, *(float (*)[4])cs); load_run<4>(p.cos + pos + 4, *(float (*)[4])(cs + 4));
        load_run<4>(p.sin + pos, *(float (*)[4])sn); load_run<4>(p.sin + pos + 4, *(float (*)[4])(sn + 4));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float ac = a[i] * cs[i], bs = b[i] * sn[i], bc = b[i] * cs[i], as = a[i] * sn[i];
            a[i] = ac - bs;
            b[i] = bc + as;
        }
        if (h < p.heads) {
            T* q = (T*)p.q + ((size_t)row * p.heads + h) * p.dim;
            store_run<4>(q + c0, *(float (*)[4])a); store_run<4>(q + c0 + 4, *(float (*)[4])(a + 4));
            store_run<4>(q + half + c0, *(float (*)[4])b); store_run<4>(q + half + c0 + 4, *(float (*)[4])(b + 4));
            return;
        }
    }
    const int slot = p.slots[row], head = h - p.heads - (value ? p.kv_heads : 0);
    cache4_put(p, slot, head, value, c0, a);
    cache4_put(p, slot, head, value, half + c0, b);
}

template <typename T, bool WORDS>
__global__ void __launch_bounds__(256)
write4_kernel(Write4Args p) {
#pragma clang fp contract(off)
    const int per_head = p.dp / 8, all = p.heads + 2 * p.kv_heads;
    const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long vector = at / per_head;
    const int u = (int)(at - vector * per_head), row = (int)(vector / all), h = (int)(vector - (long long)row * all);
    if (row >= p.rows) return;                                     // (whole blocks of 32 coordinates: their four threads leave together)
    const T* x = (const T*)p.qkv + ((size_t)row * all + h) * p.dim;
    const int c0 = 8 * u, half = p.rot / 2;
    float y[8];
    if (h >= p.heads + p.kv_heads) {
        if constexpr (WORDS) {
            if (c0 < p.dim) { load_run<4>(x + c0, *(float (*)[4])y); load_run<4>(x + c0 + 4, *(float (*)[4])(y + 4)); }
            else for (int i = 0; i < 8; ++i) y[i] = 0.f;
        } else {
            for (int i = 0; i < 8; ++i) y[i] = c0 + i < p.dim ? load_f32(x + c0 + i) : 0.f;
        }
    } else {
        const int pos = min(max(p.positions[row], 0), p.max_pos - 1);
        const float* cos = p.cos + (size_t)pos * half;
        const float* sin = p.sin + (size_t)pos * half;
        if constexpr (WORDS) {                                      // halves of whole eights: one side a thread
            if (c0 < p.rot) {
                const bool second = c0 >= half;
                const int o = second ? c0 - half : c0 + half, i0 = second ? c0 - half : c0;
                float a[8], b[8], cs[8], sn[8];
                load_run<4>(x + c0, *(float (*)[4])a); load_run<4>(x + c0 + 4, *(float (*)[4])(a + 4));
                load_run<4>(x + o, *(float (*)[4])b); load_run<4>(x + o + 4, *(float (*)[4])(b + 4));
                load_run<4>(cos + i0, *(float (*)[4])cs); load_run<4>(cos + i0 + 4, *(float (*)[4])(cs + 4));
                load_run<4>(sin + i0, *(float (*)[4])sn); load_run<4>(sin + i0 + 4, *(float (*)[4])(sn + 4));
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float ac = a[i] * cs[i], bs = b[i] * sn[i];
                    y[i] = second ? ac + bs : ac - bs;
                }
            } else if (c0 < p.dim) {
                load_run<4>(x + c0, *(float (*)[4])y); load_run<4>(x + c0 + 4, *(float (*)[4])(y + 4));
            } else {
                for (int i = 0; i < 8; ++i) y[i] = 0.f;
            }
        } else {
            for (int i = 0; i < 8; ++i) {
                const int c = c0 + i;
                if (c >= p.dim) { y[i] = 0.f; continue; }
                const float a = load_f32(x + c);
                if (c >= p.rot) { y[i] = a; continue; }
                const bool second = p.interleaved ? c & 1 : c >= half;
                const int j = p.interleaved ? c / 2 : second ? c - half : c;
                const float b = load_f32(x + (p.interleaved ? c ^ 1 : second ? c - half : c + half));
                const float ac = a * cos[j], bs = b * sin[j];
                y[i] = second ? ac + bs : ac - bs;
            }
        }
    }
    if (h < p.heads) {
        T* q = (T*)p.q + ((size_t)row * p.heads + h) * p.dim;
        if constexpr (WORDS) {
            if (c0 < p.dim) { store_run<4>(q + c0, *(float (*)[4])y); store_run<4>(q + c0 + 4, *(float (*)[4])(y + 4)); }
        } else {
            for (int i = 0; i < 8; ++i) if (c0 + i < p.dim) store_f32(q + c0 + i, y[i]);
        }
        return;
    }
    const bool value = h >= p.heads + p.kv_heads;
    cache4_put(p, p.slots[row], h - p.heads - (value ? p.kv_heads : 0), value, c0, y);
}

// What is held for the token slots `slots`, as bf16 (every held number is one).  A thread has 8 coordinates; a slot that is none gives zeros.
// Bound by the bytes that it writes: 4 sites of 4,096 tokens of 8 heads of 128, 67 MB, in 21 us.
__device__ __forceinline__ uint4 cache4_eight(uint32_t word, int s) {
    typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;
    const float scale = __uint_as_float((uint32_t)s << 23);
    uint4 r;
    r.x = __builtin_bit_cast(uint32_t, (bf16x2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 0));
    r.y = __builtin_bit_cast(uint32_t, (bf16x2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 1));
    r.z = __builtin_bit_cast(uint32_t, (bf16x2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 2));
    r.w = __builtin_bit_cast(uint32_t, (bf16x2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 3));
    return r;
}

struct Read4Args {
    const uint8_t* pages; const int* slots; bf16_t* keys; bf16_t* values;
    uint32_t pieces;                         // of a site: rows * heads * (keys, values) * eights of coordinates
    int rows, kv_heads, dim, dp, shift, n_pages;
};

__global__ void __launch_bounds__(256)
read4_kernel(Read4Args p) {
    const uint32_t per_head = (uint32_t)(p.dim + 7) / 8, at = blockIdx.x * 256 + threadIdx.x;
    if (at >= p.pieces) return;
    const uint32_t vector = at / per_head, pair = vector / p.kv_heads, site = blockIdx.y;
    const int c0 = 8 * (int)(at - vector * per_head), head = (int)(vector - pair * p.kv_heads);
    const bool value = pair >= (uint32_t)p.rows;                   // (all keys first: a wave does one thing)
    const int row = (int)(value ? pair - p.rows : pair), slot = p.slots[row];
    uint4 w = make_uint4(0, 0, 0, 0);
    if (slot >= 0 && slot >> p.shift < p.n_pages) {
        const int t = slot & ((1 << p.shift) - 1);
        const uint8_t* page = p.pages + (((size_t)site * p.n_pages + (slot >> p.shift)) * p.kv_heads + head) * cache4_record(p.dp, 1 << p.shift);
        uint32_t word = 0;
        const int width = cache4_cut(p.dp) / 16;
        if (!value) word = *(const uint32_t*)(page + cache4_key_at(p.dp, t, c0));
        else if (width == 8) word = *(const uint32_t*)(page + cache4_value_at(p.dp, p.shift, t, c0));
        else if (width == 4) for (int i = 0; i < 2; ++i) word |= (uint32_t)*(const uint16_t*)(page + cache4_value_at(p.dp, p.shift, t, c0 + 4 * i)) << (16 * i);
        else for (int i = 0; i < 4; ++i) word |= (uint32_t)page[cache4_value_at(p.dp, p.shift, t, c0 + 2 * i)] << (8 * i);
        w = cache4_eight(word, page[cache4_scale_at(p.dp, p.shift, t, c0 / 32, value)]);
    }
    bf16_t* out = (value ? p.values : p.keys) + (((size_t)site * p.rows + row) * p.kv_heads + head) * p.dim + c0;
    if (p.dim % 8 == 0) {
        *(uint4*)out = w;
    } else {
        const uint32_t words[4] = {w.x, w.y, w.z, w.w};
        for (int i = 0; i < 8 && c0 + i < p.dim; ++i) out[i] = (bf16_t)(words[i / 2] >> (16 * (i & 1)));
    }
}

// Which keys stay: of n the last `recent`, and of those before them the ones with the largest weights, as many as fill `keep`; of equal weights
// the one that came first.  A block is one head of one request at one site, its weights 16 a thread in registers (longer rows: 16,384 at a time,
// read again from the second-level cache for every pass).  The least weight that stays is found digit by digit of eight bits, from
// the first bit in which any two differ: the digits then spread over the counters, where those of whole floats would all meet at a few
// (a float's order is that of its bits, turned round for negative ones; a NaN is the least).  Then the kept indices and weights go out in
// order, their places from counts by wave and turn.  What the block has to agree on is found by every wave for itself from counters in LDS, so that a pass and
// a 16,384 cost one meeting each.  Bound by that chain: 14 us for 90 heads of 2,112 keys, 21 for 128 of up to 16,384 (18 and 26 with four meetings a pass,
// one counter a digit and a branch round each load).
// The weights may be moved within their own row: a kept one never moves up, and a 16,384 is read whole before any of it is written.
struct Evict4Args {
    const int* lengths; const int* slots; const int* new_slots; const int* tables; const int* new_tables;
    uint8_t* pages; int* kept;
    long long n_pages;
    int requests, kv_heads, dp, shift, width, new_width, keep, recent, capacity, n_slots, sites;
    float* weights[CACHE4_SITES];
};

__device__ __forceinline__ uint32_t weight_order(float w) {
    if (w != w) return 0u;
    const uint32_t b = __float_as_uint(w == 0.f ? 0.f : w);        // (both zeros are alike)
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float weight_of(uint32_t k) { return k == 0u ? NAN : __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

#define EVICT_HOLD 16
#define EVICT_COPIES 4
// The sum over this lane and those below it, without LDS: within rows of 16 lanes, then over the rows.
__device__ __forceinline__ uint32_t wave_prefix(uint32_t x) {
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, true);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, true);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, true);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, true);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, false);
    return x + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, false);
}
// How many lanes below this one are set.
__device__ __forceinline__ int lanes_below(unsigned long long set) {
    return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(set >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)set, 0u));
}
// Digits' counts of one pass as each wave takes them (four a lane): the digit whose entries reach `take` from the top, how many are of larger ones, how many its own.
struct EvictDigit { uint32_t digit, above, here; };
__device__ __forceinline__ EvictDigit evict_digit(const uint32_t (&bins)[256 * EVICT_COPIES], int lane, uint32_t take) {
    uint4 of;
    uint32_t* each = &of.x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint4 x = *(const uint4*)&bins[EVICT_COPIES * (4 * lane + j)];
        each[j] = x.x + x.y + x.z + x.w;
    }
    const uint32_t sum = of.x + of.y + of.z + of.w, up = wave_prefix(sum);
    const uint32_t over = (uint32_t)__builtin_amdgcn_readlane((int)up, WAVE - 1) - up + sum;      // of this lane's digits and larger ones
    uint32_t larger = over - sum, j = 3, here = of.w;
    if (larger + of.w < take) { larger += of.w; j = 2; here = of.z;
        if (larger + of.z < take) { larger += of.z; j = 1; here = of.y;
            if (larger + of.y < take) { larger += of.y; j = 0; here = of.x; } } }
    const int owner = __ffsll(__ballot(over >= take && over - sum < take)) - 1;      // (one lane: 0 < take <= all entries)
    return {(uint32_t)__builtin_amdgcn_readlane((int)(4 * lane + j), owner), (uint32_t)__builtin_amdgcn_readlane((int)larger, owner),
            (uint32_t)__builtin_amdgcn_readlane((int)here, owner)};
}

template <int EVICT_THREADS>
__global__ void __launch_bounds__(EVICT_THREADS)
evict4_select(Evict4Args p) {
    constexpr int WAVES = EVICT_THREADS / WAVE, SPAN = EVICT_HOLD * EVICT_THREADS, N = EVICT_HOLD * WAVES / WAVE;
    static_assert(N == 1 || N == 4, "a wave takes all counts, one or four a lane");
    __shared__ __attribute__((aligned(16))) uint32_t bins[4][256 * EVICT_COPIES];
    __shared__ uint32_t ends[2][WAVES];               // (a pass has its own counters: no meeting to clear them; four for each digit, as most entries share a few)
    __shared__ __attribute__((aligned(16))) uint32_t counts[2][EVICT_HOLD * WAVES];              // [turn][wave]: entries above `least`, and 65,536 times those at it
    const int head = blockIdx.x % p.kv_heads, request = blockIdx.x / p.kv_heads, site = blockIdx.y, tid = threadIdx.x;
    const int lane = tid % WAVE, wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
    const int from = p.slots[request], to = p.new_slots[request];
    int n = (int)min((long long)min(p.lengths[request], p.capacity), (long long)p.width << p.shift);
    if (from < 0 || from >= p.n_slots || to < 0 || to >= p.n_slots) n = 0;
    float* base = p.weights[site];
    const float* w = base + ((size_t)max(from, 0) * p.kv_heads + head) * p.capacity;
    float* nw = base + ((size_t)max(to, 0) * p.kv_heads + head) * p.capacity;
    int* kept = p.kept + (((size_t)site * p.requests + request) * p.kv_heads + head) * p.keep;
    if (n <= 0) {
        for (int i = tid; i < p.keep; i += EVICT_THREADS) kept[i] = -1;
        return;
    }
    const int old = max(0, n - p.recent);                           // these are ranked
    int take = n <= p.keep ? old : p.keep - (n - old);              // and so many of them stay
    const bool all = take >= old;
    uint32_t k[EVICT_HOLD];
    auto load = [&](int i0) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < EVICT_HOLD; ++j) {
            const int i = i0 + j * EVICT_THREADS + tid;
            k[j] = __float_as_uint(w[min(i, n - 1)]);               // (no branch round a load: all are on their way together)
        }
#pragma unroll
        for (int j = 0; j < EVICT_HOLD; ++j) k[j] = weight_order(__uint_as_float(k[j]));
    };
    load(0);
    uint32_t least = 0;                                             // kept: above `least`, and the first `take` at it
    if (!all && take > 0) {
        // the smallest and the largest of the ranked
        uint32_t low = 0xffffffffu, high = 0u;
        for (int i0 = 0; i0 < old; i0 += SPAN) {
            if (i0 > 0) load(i0);
#pragma unroll
            for (int j = 0; j < EVICT_HOLD; ++j)
                if (i0 + j * EVICT_THREADS + tid < old) { low = min(low, k[j]); high = max(high, k[j]); }
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) { low = min(low, __shfl_xor(low, off, WAVE)); high = max(high, __shfl_xor(high, off, WAVE)); }
        if (lane == 0) { ends[0][wave] = low; ends[1][wave] = high; }
        for (int i = tid; i < 256 * EVICT_COPIES; i += EVICT_THREADS) ((uint4*)bins)[i] = make_uint4(0u, 0u, 0u, 0u);
        __syncthreads();
#pragma unroll
        for (int v = 0; v < WAVES; ++v) { low = min(low, ends[0][v]); high = max(high, ends[1][v]); }
        least = low;                                                // (the digits found so far, from `low` on)
        int bits = high > low ? 32 - __clz(high - low) : 0;         // that are still open
        for (int pass = 0; bits > 0; ++pass) {                      // (four at most: 32 bits in eights)
            const int shift = max(bits - 8, 0);
            for (int i0 = 0; i0 < old; i0 += SPAN) {
                if (old > SPAN) load(i0);
#pragma unroll
                for (int j = 0; j < EVICT_HOLD; ++j) {
                    if (i0 + j * EVICT_THREADS >= old) break;
                    const uint32_t d = k[j] - least;                // (below `least`: a large number)
                    if (i0 + j * EVICT_THREADS + tid < old && k[j] >= least && (bits == 32 || d >> bits == 0)) atomicAdd(&bins[pass][EVICT_COPIES * (d >> shift) + lane % EVICT_COPIES], 1u);
                }
            }
            __syncthreads();
            const EvictDigit got = evict_digit(bins[pass], lane, (uint32_t)take);
            least += got.digit << shift;
            take -= (int)got.above;
            bits = shift;
            if ((int)got.here == take) {                            // all of this digit stay: the rest of the bits say nothing
                take = 0x7fffffff;
                break;
            }
        }
        if (old > SPAN) load(0);
    } else if (!all) {
        least = 0xffffffffu;
        take = 0;
    }
    int done = 0, met = 0;                                          // entries above and at `least` of the spans before
    for (int i0 = 0, turn = 0; i0 < n; i0 += SPAN, turn ^= 1) {
        if (i0 > 0) load(i0);
        unsigned long long tie[EVICT_HOLD], over[EVICT_HOLD];
        uint32_t mine = 0;
#pragma unroll
        for (int j = 0; j < EVICT_HOLD; ++j) {
            const int i = i0 + j * EVICT_THREADS + tid;
            tie[j] = __ballot(!all && i < old && k[j] == least);
            over[j] = __ballot(i < n && (all || i >= old || k[j] > least));
            const uint32_t of = (uint32_t)(__popcll(over[j]) | __popcll(tie[j]) << 16);
            mine = lane == j ? of : mine;
        }
        if (lane < EVICT_HOLD) counts[turn][lane * WAVES + wave] = mine;
        __syncthreads();                                            // (and everyone has read its weights)
        uint32_t own[N], sum = 0;                                   // (a span has 16,384 entries: neither half runs over)
        if constexpr (N == 4) {
            const uint4 x = *(const uint4*)&counts[turn][4 * lane];
            own[0] = x.x; own[1] = x.y; own[2] = x.z; own[3] = x.w;
        } else {
            own[0] = counts[turn][lane];
        }
#pragma unroll
        for (int x = 0; x < N; ++x) { const uint32_t of = own[x]; own[x] = sum; sum += of; }
        uint32_t up = wave_prefix(sum);
        const uint32_t total = (uint32_t)__builtin_amdgcn_readlane((int)up, WAVE - 1);
        up -= sum;
        uint32_t at = own[0];                                       // before this wave's entry of the lane's N
#pragma unroll
        for (int x = 1; x < N; ++x) at = wave % N == x ? own[x] : at;
        at += up;
#pragma unroll
        for (int j = 0; j < EVICT_HOLD; ++j) {
            if (i0 + j * EVICT_THREADS >= n) break;
            const uint32_t first = (uint32_t)__builtin_amdgcn_readlane((int)at, (j * WAVES + wave) / N);
            const int ties = met + (int)(first >> 16) + lanes_below(tie[j]);
            const int place = done + (int)(first & 0xffffu) + lanes_below(over[j]) + min(ties, take);
            if ((over[j] >> lane & 1 || (tie[j] >> lane & 1 && ties < take)) && place < p.keep) { kept[place] = i0 + j * EVICT_THREADS + tid; nw[place] = weight_of(k[j]); }
        }
        done += (int)(total & 0xffffu);
        met += (int)(total >> 16);
    }
    const int m = min(done + min(met, take), p.keep);
    for (int i = m + tid; i < p.keep; i += EVICT_THREADS) kept[i] = -1;
    for (int i = m + tid; i < p.capacity; i += EVICT_THREADS) nw[i] = 0.f;
}

// The kept keys and values, from the pages that held them to the pages of the new table: a block is 64 tokens of a head.  Keys go in rows of 16-byte
// pieces; of the values a thread gathers the run of a column and eight tokens and writes it whole, likewise of the scales.  Bound by the chain kept index,
// page, bytes and by the gathered words: 30 sites of 2,048 keys of 3 heads of 64 in 12.6 us (15.7 where all three are asked for before any is written, with
// places reckoned without a branch).
#define EVICT_TOKENS 64
__global__ void __launch_bounds__(256)
evict4_move(Evict4Args p) {
    const int tiles = (p.keep + EVICT_TOKENS - 1) / EVICT_TOKENS, tid = threadIdx.x;
    const int tile = blockIdx.x % tiles, head = blockIdx.x / tiles, request = blockIdx.y, site = blockIdx.z;
    const int P = 1 << p.shift, mask = P - 1, record = cache4_record(p.dp, P), first = EVICT_TOKENS * tile;
    __shared__ const uint8_t* source[EVICT_TOKENS];                 // of a token: its page, and the page of its place; null where there is none
    __shared__ uint8_t* target[EVICT_TOKENS];
    __shared__ int token[EVICT_TOKENS];
    const int* kept = p.kept + (((size_t)site * p.requests + request) * p.kv_heads + head) * p.keep;
    uint8_t* pages = p.pages + (size_t)site * p.n_pages * p.kv_heads * record;
    if (tid < EVICT_TOKENS) {
        const int i = first + tid, k = i < p.keep ? kept[i] : -1;
        const int page = k >= 0 && k >> p.shift < p.width ? p.tables[(size_t)request * p.width + (k >> p.shift)] : -1;
        const int to = i >> p.shift < p.new_width ? p.new_tables[(size_t)request * p.new_width + (i >> p.shift)] : -1;
        source[tid] = page >= 0 && page < p.n_pages ? pages + ((size_t)page * p.kv_heads + head) * record : nullptr;
        target[tid] = to >= 0 && to < p.n_pages ? pages + ((size_t)to * p.kv_heads + head) * record : nullptr;
        token[tid] = k & mask;
    }
    __syncthreads();
    const int pieces = p.dp / 32;
    for (int i = tid; i < EVICT_TOKENS * pieces; i += 256) {
        const int t = i / pieces, x = i - t * pieces;
        if (source[t] && target[t]) *(uint4*)(target[t] + ((first + t) & mask) * (p.dp / 2) + 16 * x) = *(const uint4*)(source[t] + token[t] * (p.dp / 2) + 16 * x);
    }
    const int cut = cache4_cut(p.dp), w = cut / 16, columns = p.dp / w;
    for (int i = tid; i < EVICT_TOKENS / 8 * columns; i += 256) {
        const int e = i / columns, d = (i - e * columns) * w, t0 = 8 * e;
        if (!target[t0]) continue;                                  // (eight tokens are in one page)
        uint8_t* out = target[t0] + cache4_value_at(p.dp, p.shift, (first + t0) & mask, d);
        bool whole = true;
        uint32_t run[8];
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            const uint8_t* in = source[t0 + t] ? source[t0 + t] + cache4_value_at(p.dp, p.shift, token[t0 + t], d) : nullptr;
            whole &= in != nullptr;
            run[t] = !in ? 0u : w == 8 ? *(const uint32_t*)in : w == 4 ? *(const uint16_t*)in : *in;
        }
        if (whole && w == 8) {
            *(uint4*)out = make_uint4(run[0], run[1], run[2], run[3]);
            *(uint4*)(out + 16) = make_uint4(run[4], run[5], run[6], run[7]);
        } else if (whole && w == 4) {
            *(uint4*)out = make_uint4(run[0] | run[1] << 16, run[2] | run[3] << 16, run[4] | run[5] << 16, run[6] | run[7] << 16);
        } else if (whole) {
            *(uint2*)out = make_uint2(run[0] | run[1] << 8 | run[2] << 16 | run[3] << 24, run[4] | run[5] << 8 | run[6] << 16 | run[7] << 24);
        } else {                                                    // (what lies behind the last kept key is left as it is)
#pragma unroll
            for (int t = 0; t < 8; ++t)
                if (source[t0 + t]) {
                    if (w == 8) *(uint32_t*)(out + 4 * t) = run[t];
                    else if (w == 4) *(uint16_t*)(out + 2 * t) = (uint16_t)run[t];
                    else out[t] = (uint8_t)run[t];
                }
        }
    }
    const int blocks = p.dp / 32;
    for (int i = tid; i < EVICT_TOKENS / 8 * 2 * blocks; i += 256) {
        const int e = i / (2 * blocks), b = i - e * 2 * blocks, t0 = 8 * e;
        if (!target[t0]) continue;
        const bool value = b >= blocks;
        bool whole = true;
        uint8_t* out = target[t0] + cache4_scale_at(p.dp, p.shift, (first + t0) & mask, value ? b - blocks : b, value);
        uint32_t run[8];
#pragma unroll
        for (int t = 0; t < 8; ++t) whole &= source[t0 + t] != nullptr;
#pragma unroll
        for (int t = 0; t < 8; ++t) run[t] = source[t0 + t] ? source[t0 + t][cache4_scale_at(p.dp, p.shift, token[t0 + t], value ? b - blocks : b, value)] : 0u;
        if (whole) {
            *(uint2*)out = make_uint2(run[0] | run[1] << 8 | run[2] << 16 | run[3] << 24, run[4] | run[5] << 8 | run[6] << 16 | run[7] << 24);
        } else {
#pragma unroll
            for (int t = 0; t < 8; ++t) if (source[t0 + t]) out[t] = (uint8_t)run[t];
        }
    }
}

// Partial results of keys in several pieces: part_o [piece][key head][row of the task][head of the group][dim], part_ml likewise [2] (maximum
// in powers of two, sum).  `merges` [n][4]: first row (negative: none), rows, first piece, pieces.  Bound by the launch and two trips to memory: 4 us.
struct Merge4Args {
    const float* part_o; const float* part_ml; const int* merges; void* out; float* stats;
    int rows_per_task, heads, kv_heads, group, dim;
};

template <typename T>
__global__ void __launch_bounds__(256)
merge4_kernel(Merge4Args p) {
    const int* list = p.merges + 4 * (size_t)blockIdx.x;
    const int row0 = list[0], rows = list[1], first = list[2], pieces = list[3], halves = p.dim / 2;
    if (row0 < 0) return;
    const int at = blockIdx.y * 256 + threadIdx.x, item = at / halves, d = 2 * (at - item * halves);    // (item: row, head)
    if (item >= rows * p.heads) return;
    const int r = item / p.heads, h = item - r * p.heads, kvh = h / p.group;
    const size_t one = ((size_t)kvh * p.rows_per_task + r) * p.group + h - kvh * p.group, step = (size_t)p.heads * p.rows_per_task;
    // (eight pieces' loads are on their way together: one trip to memory instead of one a piece)
    float m = CACHE4_NOTHING, l = 0.f, a = 0.f, b = 0.f;
    for (int s0 = 0; s0 < pieces; s0 += 8) {
        float2 ml[8], v[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            const size_t part = (first + min(s0 + s, pieces - 1)) * step + one;
            ml[s] = *(const float2*)(p.part_ml + 2 * part);
            v[s] = *(const float2*)(p.part_o + part * p.dim + d);
        }
        float top = m;
#pragma unroll
        for (int s = 0; s < 8; ++s) top = s0 + s < pieces ? fmaxf(top, ml[s].x) : top;
        const float f = exp2f(m - top);
        m = top;
        l *= f;
        a *= f;
        b *= f;
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            const float g = s0 + s < pieces ? exp2f(ml[s].x - top) : 0.f;
            l = fmaf(ml[s].y, g, l);
            a = fmaf(v[s].x, g, a);
            b = fmaf(v[s].y, g, b);
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const size_t to = (size_t)(row0 + r) * p.heads + h;
    if constexpr (sizeof(T) == 4) *(float2*)((float*)p.out + to * p.dim + d) = make_float2(a * inv, b * inv);
    else *(uint32_t*)((bf16_t*)p.out + to * p.dim + d) = pack_bf16x2(a * inv, b * inv);
    if (p.stats && d == 0) p.stats[to] = m + log2f(l);
}

// What an entry point is called with, one block of bytes (a pointer to it is converted in a tenth of the time of 20 arguments, 1 us of 9 a call).
struct Write4Call {
    hipStream_t stream; const void* qkv; const int* positions; const int* slots; const float* cos; const float* sin; uint8_t* pages; void* q;
    int rows, heads, kv_heads, dim, rot, page, n_pages, max_pos, interleaved, dtype;
};
struct Read4Call { hipStream_t stream; const uint8_t* pages; const int* slots; bf16_t* keys; bf16_t* values; int sites, rows, kv_heads, dim, page, n_pages; };
struct Evict4Call {
    hipStream_t stream; const int* lengths; const int* slots; const int* new_slots; const int* tables; const int* new_tables; uint8_t* pages; int* kept;
    int sites, n_pages, requests, kv_heads, dim, page, width, new_width, keep, recent, capacity, n_slots;
};
struct Merge4Call { hipStream_t stream; const float* part_o; const float* part_ml; const int* merges; void* out; float* stats; int n, rows_per_task, heads, kv_heads, dim, dtype; };

extern "C" {

// Bytes of a call as it is here, by entry point: what the caller packs has to agree.
int cisr_call4_bytes(int which) {
    const size_t bytes[] = {sizeof(Write4Call), sizeof(Read4Call), sizeof(Evict4Call), sizeof(Merge4Call), sizeof(Attn4Call), sizeof(Weights4Call)};
    return which >= 0 && which < 6 ? (int)bytes[which] : -1;
}

int cisr_write4(const Write4Call* call) {
    const auto [stream, qkv, positions, slots, cos, sin, pages, q, rows, heads, kv_heads, dim, rot, page, n_pages, max_pos, interleaved, dtype] = *call;
    if (rows <= 0 || heads <= 0 || kv_heads <= 0 || dim <= 0 || dim > 256 || dim % 2 || rot < 0 || rot > dim || rot % 2 || page < 8 || (page & (page - 1)) || n_pages <= 0 || max_pos <= 0)
        return hipErrorInvalidValue;
    const int dp = (dim + 31) / 32 * 32;
    Write4Args p = {qkv, positions, slots, cos, sin, (uint8_t*)pages, q, rows, heads, kv_heads, dim, dp, rot, __builtin_ctz(page), max_pos, n_pages, interleaved};
    const long long blocks = ((long long)rows * (heads + 2 * kv_heads) * (dp / 8) + 255) / 256;
    if (blocks > INT32_MAX / 256) return hipErrorInvalidValue;
    const uintptr_t both = (uintptr_t)qkv | (uintptr_t)q | (uintptr_t)cos | (uintptr_t)sin;
    const bool words = !interleaved && dim % 8 == 0 && rot % 16 == 0 && both % 16 == 0;
    if (words && rot == dim && dim % 64 == 0) {
        const int half_blocks = (int)(((long long)rows * (heads + 2 * kv_heads) * (dim / 16) + 255) / 256);
        if (dtype == DT_BF16) write4_halves_kernel<bf16_t><<<half_blocks, 256, 0, (hipStream_t)stream>>>(p);
        else write4_halves_kernel<float><<<half_blocks, 256, 0, (hipStream_t)stream>>>(p);
    } else if (dtype == DT_BF16) {
        if (words) write4_kernel<bf16_t, true><<<(int)blocks, 256, 0, (hipStream_t)stream>>>(p);
        else write4_kernel<bf16_t, false><<<(int)blocks, 256, 0, (hipStream_t)stream>>>(p);
    } else {
        if (words) write4_kernel<float, true><<<(int)blocks, 256, 0, (hipStream_t)stream>>>(p);
        else write4_kernel<float, false><<<(int)blocks, 256, 0, (hipStream_t)stream>>>(p);
    }
    return hipGetLastError();
}

int cisr_read4(const Read4Call* call) {
    const auto [stream, pages, slots, keys, values, sites, rows, kv_heads, dim, page, n_pages] = *call;
    if (sites <= 0 || rows <= 0 || kv_heads <= 0 || dim <= 0 || dim > 256 || dim % 2 || page < 8 || (page & (page - 1)) || n_pages <= 0) return hipErrorInvalidValue;
    const long long pieces = (long long)rows * kv_heads * 2 * ((dim + 7) / 8);
    if (pieces > INT32_MAX || sites > 65535) return hipErrorInvalidValue;
    Read4Args p = {(const uint8_t*)pages, slots, (bf16_t*)keys, (bf16_t*)values, (uint32_t)pieces, rows, kv_heads, dim, (dim + 31) / 32 * 32, __builtin_ctz(page), n_pages};
    read4_kernel<<<dim3((uint32_t)((pieces + 255) / 256), sites), 256, 0, (hipStream_t)stream>>>(p);
    return hipGetLastError();
}

int cisr_evict4(const Evict4Call* call, void* const* weights) {
    const auto [stream, lengths, slots, new_slots, tables, new_tables, pages, kept, sites, n_pages, requests, kv_heads, dim, page, width, new_width, keep, recent, capacity,
                n_slots] = *call;
    if (sites <= 0 || n_pages <= 0 || requests <= 0 || requests > 65535 || kv_heads <= 0 || dim <= 0 || dim > 256 || page < 8 || (page & (page - 1)) || width <= 0 || new_width <= 0 || keep <= 0 ||
        recent < 0 || recent > keep || capacity < keep || n_slots <= 0)
        return hipErrorInvalidValue;
    const int dp = (dim + 31) / 32 * 32;
    const size_t site_bytes = (size_t)n_pages * kv_heads * cache4_record(dp, page);
    for (int at = 0; at < sites; at += CACHE4_SITES) {              // (the sites' weights travel with the launch)
        const int now = sites - at < CACHE4_SITES ? sites - at : CACHE4_SITES;
        Evict4Args p = {lengths, slots, new_slots, tables, new_tables, (uint8_t*)pages + at * site_bytes, kept + (size_t)at * requests * kv_heads * keep, n_pages,
                        requests, kv_heads, dp, __builtin_ctz(page), width, new_width, keep, recent, capacity, n_slots, now, {}};
        for (int s = 0; s < now; ++s) p.weights[s] = (float*)weights[at + s];
        // (blocks of four waves meet faster, and hold rows of up to 4,096)
        if ((capacity < (long long)width * page ? capacity : (long long)width * page) <= 256 * EVICT_HOLD) evict4_select<256><<<dim3(requests * kv_heads, now), 256, 0, (hipStream_t)stream>>>(p);
        else evict4_select<1024><<<dim3(requests * kv_heads, now), 1024, 0, (hipStream_t)stream>>>(p);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        evict4_move<<<dim3((keep + EVICT_TOKENS - 1) / EVICT_TOKENS * kv_heads, requests, now), 256, 0, (hipStream_t)stream>>>(p);
        e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

int cisr_merge4(const Merge4Call* call) {
    const auto [stream, part_o, part_ml, merges, out, stats, n, rows_per_task, heads, kv_heads, dim, dtype] = *call;
    if (n <= 0 || rows_per_task <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || dim <= 0 || dim % 2) return hipErrorInvalidValue;
    const long long blocks = ((long long)rows_per_task * heads * (dim / 2) + 255) / 256;
    if (blocks > 65535) return hipErrorInvalidValue;
    Merge4Args p = {part_o, part_ml, merges, out, stats, rows_per_task, heads, kv_heads, heads / kv_heads, dim};
    if (dtype == DT_BF16) merge4_kernel<bf16_t><<<dim3(n, (int)blocks), 256, 0, (hipStream_t)stream>>>(p);
    else merge4_kernel<float><<<dim3(n, (int)blocks), 256, 0, (hipStream_t)stream>>>(p);
    return hipGetLastError();
}

}  // extern "C"
