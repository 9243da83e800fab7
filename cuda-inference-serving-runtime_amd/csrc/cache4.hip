// Writing into the cache that is held in 4 bits, reading it back, and giving up the keys with the least attention weight.
//
// Write: q' = rot(q) goes to rows of its own, rot(k) and v to the pages.  A thread has 8 coordinates, four threads a block; the
// block's scale follows from its largest magnitude a alone: 2^s with a / 2^s in (3.5, 7], which is the exponent of a after
// a quarter of its leading bit has been added (normal numbers: 11.2 % off; the limits 6 and 8 give 11.5 %).  The rotary sums are rounded
// product by product, without fused steps, so that a code near a border does not depend on how a compiler joins them.
// An infinity is held as the largest number of the largest scale, a NaN as zero: what is cached is always finite.
// Bound by the bytes of the rows.
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
    const float inv = __uint_as_float((uint32_t)(127 - s) << 23);
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float y = fabsf(x[i]) * inv;
        const uint32_t code = (y > 0.25f) + (y >= 0.75f) + (y > 1.25f) + (y >= 1.75f) + (y > 2.5f) + (y >= 3.5f) + (y > 5.f);
        word |= (code | (x[i] < 0.f ? 8u : 0u)) << (4 * i);
    }
    return word;
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
    const int slot = p.slots[row];
    const bool value = h >= p.heads + p.kv_heads;
    const int head = h - p.heads - (value ? p.kv_heads : 0);
    int s;
    const uint32_t word = cache4_codes(y, s);
    if (slot < 0 || slot >> p.shift >= p.n_pages) return;
    const int t = slot & ((1 << p.shift) - 1);
    uint8_t* page = p.pages + ((size_t)(slot >> p.shift) * p.kv_heads + head) * cache4_record(p.dp, 1 << p.shift);
    if ((u & 3) == 0) page[cache4_scale_at(p.dp, p.shift, t, u / 4, value)] = (uint8_t)(s + CACHE4_BIAS);
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

// What is held for the token slots `slots`, as bf16 (every held number is one).  A thread has 8 coordinates; a slot that is none gives zeros.
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
    long long vectors;                       // sites * rows * heads * 2
    int rows, kv_heads, dim, dp, shift, n_pages;
};

__global__ void __launch_bounds__(256)
read4_kernel(Read4Args p) {
    const int per_head = (p.dim + 7) / 8;
    const long long at = (long long)blockIdx.x * 256 + threadIdx.x, vector = at / per_head;
    if (vector >= p.vectors) return;
    const int c0 = 8 * (int)(at - vector * per_head), head = (int)(vector % p.kv_heads);
    long long rest = vector / p.kv_heads;
    const int row = (int)(rest % p.rows);
    rest /= p.rows;
    const bool value = rest & 1;
    const long long site = rest >> 1;
    const int slot = p.slots[row];
    uint4 w = make_uint4(0, 0, 0, 0);
    if (slot >= 0 && slot >> p.shift < p.n_pages) {
        const int t = slot & ((1 << p.shift) - 1);
        const uint8_t* page = p.pages + ((size_t)(site * p.n_pages + (slot >> p.shift)) * p.kv_heads + head) * cache4_record(p.dp, 1 << p.shift);
        uint32_t word = 0;
        const int width = cache4_cut(p.dp) / 16;
        if (!value) word = *(const uint32_t*)(page + cache4_key_at(p.dp, t, c0));
        else if (width == 8) word = *(const uint32_t*)(page + cache4_value_at(p.dp, p.shift, t, c0));
        else if (width == 4) for (int i = 0; i < 2; ++i) word |= (uint32_t)*(const uint16_t*)(page + cache4_value_at(p.dp, p.shift, t, c0 + 4 * i)) << (16 * i);
        else for (int i = 0; i < 4; ++i) word |= (uint32_t)page[cache4_value_at(p.dp, p.shift, t, c0 + 2 * i)] << (8 * i);
        w = cache4_eight(word, page[cache4_scale_at(p.dp, p.shift, t, c0 / 32, value)]);
    }
    bf16_t* out = (value ? p.values : p.keys) + ((size_t)(site * p.rows + row) * p.kv_heads + head) * p.dim + c0;
    if (p.dim % 8 == 0) {
        *(uint4*)out = w;
    } else {
        const uint32_t words[4] = {w.x, w.y, w.z, w.w};
        for (int i = 0; i < 8 && c0 + i < p.dim; ++i) out[i] = (bf16_t)(words[i / 2] >> (16 * (i & 1)));
    }
}

// Which keys stay: of n the last `recent`, and of those before them the ones with the largest weights, as many as fill `keep`; of equal weights
// the one that came first.  A block is one head of one request at one site.  The least weight that stays is found digit by digit of eight bits
// (a float's order is that of its bits, turned round for negative ones; a NaN is the least); then one pass from the front writes the kept
// indices and weights in order.  Both passes read the weights again from the second-level cache, which holds them.
// The weights may be moved within their own row: a kept one never moves up, and a piece is read whole before any of it is written.
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

#define EVICT_THREADS 1024
__global__ void __launch_bounds__(EVICT_THREADS)
evict4_select(Evict4Args p) {
    constexpr int WAVES = EVICT_THREADS / WAVE;
    __shared__ uint32_t bins[256], below[256];
    __shared__ uint32_t digit, above;
    __shared__ int larger[2][WAVES], equal[2][WAVES];
    const int head = blockIdx.x % p.kv_heads, request = blockIdx.x / p.kv_heads, site = blockIdx.y, tid = threadIdx.x;
    const int from = p.slots[request], to = p.new_slots[request];
    int n = min(min(p.lengths[request], p.capacity), p.width << p.shift);
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
    uint32_t least = 0;                                             // kept: above `least`, and the first `take` at it
    if (take < old) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) bins[tid] = 0;
            __syncthreads();
            const uint32_t mask = shift == 24 ? 0u : ~0u << (shift + 8);
            for (int i = tid; i < old; i += EVICT_THREADS) {
                const uint32_t k = weight_order(w[i]);
                if ((k & mask) == least) atomicAdd(&bins[(k >> shift) & 255], 1u);
            }
            __syncthreads();
            // entries of a larger digit, by a sum from the top over one wave: four digits a lane
            if (tid < WAVE) {
                uint32_t own[4], sum = 0;
#pragma unroll
                for (int j = 3; j >= 0; --j) { own[j] = sum; sum += bins[4 * tid + j]; }
                uint32_t over = sum;
#pragma unroll
                for (int off = 1; off < WAVE; off <<= 1) {
                    const uint32_t up = __shfl_down(over, off, WAVE);
                    if (tid + off < WAVE) over += up;
                }
                over -= sum;                                        // of the lanes above
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t more = over + own[j], here = bins[4 * tid + j];
                    if (more < (uint32_t)take && more + here >= (uint32_t)take) { digit = 4 * tid + j; above = more; }
                }
                if (tid == 0 && take <= 0) { digit = 255; above = 0; }
            }
            __syncthreads();
            least |= digit << shift;
            take -= (int)above;
            __syncthreads();
        }
    } else {
        take = 0;
    }
    const bool all = n <= p.keep || p.keep - (n - old) >= old;
    // (of those at `least` the first `take` stay)
    const int lane = tid % WAVE, wave = tid / WAVE;
    int done = 0, met = 0, turn = 0;
    for (int i0 = 0; i0 < n; i0 += EVICT_THREADS, turn ^= 1) {
        const int i = i0 + tid;
        const float weight = i < n ? w[i] : 0.f;
        const uint32_t k = weight_order(weight);
        const bool ranked = i < old && !all;
        const bool tie = ranked && k == least;
        const unsigned long long ties = __ballot(tie);
        if (lane == 0) equal[turn][wave] = __popcll(ties);
        __syncthreads();                                            // (and everyone has read its weight)
        int tied = met + __popcll(ties & ((1ull << lane) - 1)), ties_all = 0;
#pragma unroll
        for (int v = 0; v < WAVES; ++v) { const int e = equal[turn][v]; tied += v < wave ? e : 0; ties_all += e; }
        const bool stays = i < n && (!ranked || k > least || (tie && tied < take));
        const unsigned long long stay = __ballot(stays);
        if (lane == 0) larger[turn][wave] = __popcll(stay);
        __syncthreads();
        int to_index = done + __popcll(stay & ((1ull << lane) - 1)), all_stay = 0;
#pragma unroll
        for (int v = 0; v < WAVES; ++v) { const int e = larger[turn][v]; to_index += v < wave ? e : 0; all_stay += e; }
        if (stays && to_index < p.keep) { kept[to_index] = i; nw[to_index] = weight; }
        done += all_stay;
        met += ties_all;
    }
    __syncthreads();
    const int m = min(done, p.keep);
    for (int i = m + tid; i < p.keep; i += EVICT_THREADS) kept[i] = -1;
    for (int i = m + tid; i < p.capacity; i += EVICT_THREADS) nw[i] = 0.f;
}

// The kept keys and values, from the pages that held them to the pages of the new table: a block is eight tokens of a head.
__global__ void __launch_bounds__(256)
evict4_move(Evict4Args p) {
    const int eights = (p.keep + 7) / 8, tid = threadIdx.x;
    const int eight = blockIdx.x % eights, head = blockIdx.x / eights, request = blockIdx.y, site = blockIdx.z;
    const int P = 1 << p.shift, record = cache4_record(p.dp, P), first = 8 * eight;
    __shared__ const uint8_t* source[8];
    __shared__ int token[8];
    const int* kept = p.kept + (((size_t)site * p.requests + request) * p.kv_heads + head) * p.keep;
    uint8_t* site_pages = p.pages + (size_t)site * p.n_pages * p.kv_heads * record;
    const int to = first >> p.shift < p.new_width ? p.new_tables[(size_t)request * p.new_width + (first >> p.shift)] : -1;
    if (tid < 8) {
        const int k = first + tid < p.keep ? kept[first + tid] : -1;
        const int page = k >= 0 ? p.tables[(size_t)request * p.width + (k >> p.shift)] : -1;
        source[tid] = page >= 0 && page < p.n_pages ? site_pages + ((size_t)page * p.kv_heads + head) * record : nullptr;
        token[tid] = k & (P - 1);
    }
    __syncthreads();
    if (to < 0 || to >= p.n_pages) return;
    uint8_t* target = site_pages + ((size_t)to * p.kv_heads + head) * record;
    const int words = p.dp / 8, w = cache4_cut(p.dp) / 16;          // 4-byte words a token's key
    for (int i = tid; i < 8 * words; i += 256) {
        const int t = i / words, x = i % words;
        if (source[t]) *(uint32_t*)(target + ((first & (P - 1)) + t) * (p.dp / 2) + 4 * x) = *(const uint32_t*)(source[t] + token[t] * (p.dp / 2) + 4 * x);
    }
    // values: pieces of w / 2 bytes, the eight tokens side by side
    const int pieces = p.dp / w;
    for (int i = tid; i < 8 * pieces; i += 256) {
        const int t = i & 7, d = (i >> 3) * w;
        if (!source[t]) continue;
        uint8_t* out = target + cache4_value_at(p.dp, p.shift, (first & (P - 1)) + t, d);
        const uint8_t* in = source[t] + cache4_value_at(p.dp, p.shift, token[t], d);
        if (w == 8) *(uint32_t*)out = *(const uint32_t*)in;
        else if (w == 4) *(uint16_t*)out = *(const uint16_t*)in;
        else *out = *in;
    }
    const int scales = 2 * (p.dp / 32);
    for (int i = tid; i < 8 * scales; i += 256) {
        const int t = i & 7, b = i >> 3, blocks = p.dp / 32;
        if (source[t])
            target[cache4_scale_at(p.dp, p.shift, (first & (P - 1)) + t, b % blocks, b >= blocks)] = source[t][cache4_scale_at(p.dp, p.shift, token[t], b % blocks, b >= blocks)];
    }
}

// Partial results of keys in several pieces: part_o [piece][key head][row of the task][head of the group][dim], part_ml likewise [2] (maximum
// in powers of two, sum).  `merges` [n][4]: first row (negative: none), rows, first piece, pieces.
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
    float m = CACHE4_NOTHING, l = 0.f, a = 0.f, b = 0.f;
    for (int s = 0; s < pieces; ++s) {
        const size_t part = (first + s) * step + one;
        const float2 ml = *(const float2*)(p.part_ml + 2 * part), v = *(const float2*)(p.part_o + part * p.dim + d);
        const float top = fmaxf(m, ml.x), f = exp2f(m - top), g = exp2f(ml.x - top);
        m = top;
        l = fmaf(ml.y, g, l * f);
        a = fmaf(v.x, g, a * f);
        b = fmaf(v.y, g, b * f);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const size_t to = (size_t)(row0 + r) * p.heads + h;
    if constexpr (sizeof(T) == 4) *(float2*)((float*)p.out + to * p.dim + d) = make_float2(a * inv, b * inv);
    else *(uint32_t*)((bf16_t*)p.out + to * p.dim + d) = pack_bf16x2(a * inv, b * inv);
    if (p.stats && d == 0) p.stats[to] = m + log2f(l);
}

extern "C" {

int cisr_write4(const void* qkv, const int* positions, const int* slots, const float* cos, const float* sin, void* pages, void* q, int rows, int heads,
                int kv_heads, int dim, int rot, int page, int n_pages, int max_pos, int interleaved, int dtype, void* stream) {
    if (rows <= 0 || heads <= 0 || kv_heads <= 0 || dim <= 0 || dim > 256 || dim % 2 || rot < 0 || rot > dim || rot % 2 || page < 8 || (page & (page - 1)) || n_pages <= 0 || max_pos <= 0)
        return hipErrorInvalidValue;
    const int dp = (dim + 31) / 32 * 32;
    Write4Args p = {qkv, positions, slots, cos, sin, (uint8_t*)pages, q, rows, heads, kv_heads, dim, dp, rot, __builtin_ctz(page), max_pos, n_pages, interleaved};
    const long long blocks = ((long long)rows * (heads + 2 * kv_heads) * (dp / 8) + 255) / 256;
    if (blocks > INT32_MAX) return hipErrorInvalidValue;
    const uintptr_t both = (uintptr_t)qkv | (uintptr_t)q | (uintptr_t)cos | (uintptr_t)sin;
    const bool words = !interleaved && dim % 8 == 0 && rot % 16 == 0 && both % 16 == 0;
    if (dtype == DT_BF16) {
        if (words) write4_kernel<bf16_t, true><<<(int)blocks, 256, 0, (hipStream_t)stream>>>(p);
        else write4_kernel<bf16_t, false><<<(int)blocks, 256, 0, (hipStream_t)stream>>>(p);
    } else {
        if (words) write4_kernel<float, true><<<(int)blocks, 256, 0, (hipStream_t)stream>>>(p);
        else write4_kernel<float, false><<<(int)blocks, 256, 0, (hipStream_t)stream>>>(p);
    }
    return hipGetLastError();
}

int cisr_read4(const void* pages, const int* slots, void* keys, void* values, int sites, int rows, int kv_heads, int dim, int page, int n_pages, void* stream) {
    if (sites <= 0 || rows <= 0 || kv_heads <= 0 || dim <= 0 || dim > 256 || dim % 2 || page < 8 || (page & (page - 1)) || n_pages <= 0) return hipErrorInvalidValue;
    Read4Args p = {(const uint8_t*)pages, slots, (bf16_t*)keys, (bf16_t*)values, (long long)sites * rows * kv_heads * 2, rows, kv_heads, dim, (dim + 31) / 32 * 32,
                   __builtin_ctz(page), n_pages};
    const long long blocks = (p.vectors * ((dim + 7) / 8) + 255) / 256;
    if (blocks > INT32_MAX) return hipErrorInvalidValue;
    read4_kernel<<<(int)blocks, 256, 0, (hipStream_t)stream>>>(p);
    return hipGetLastError();
}

int cisr_evict4(const int* lengths, const int* slots, const int* new_slots, const int* tables, const int* new_tables, void* pages, void* const* weights, int* kept,
                int sites, int n_pages, int requests, int kv_heads, int dim, int page, int width, int new_width, int keep, int recent, int capacity, int n_slots, void* stream) {
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
        evict4_select<<<dim3(requests * kv_heads, now), EVICT_THREADS, 0, (hipStream_t)stream>>>(p);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        evict4_move<<<dim3((keep + 7) / 8 * kv_heads, requests, now), 256, 0, (hipStream_t)stream>>>(p);
        e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

int cisr_merge4(const float* part_o, const float* part_ml, const int* merges, void* out, float* stats, int n, int rows_per_task, int heads, int kv_heads, int dim, int dtype,
                void* stream) {
    if (n <= 0 || rows_per_task <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || dim <= 0 || dim % 2) return hipErrorInvalidValue;
    const long long blocks = ((long long)rows_per_task * heads * (dim / 2) + 255) / 256;
    if (blocks > 65535) return hipErrorInvalidValue;
    Merge4Args p = {part_o, part_ml, merges, out, stats, rows_per_task, heads, kv_heads, heads / kv_heads, dim};
    if (dtype == DT_BF16) merge4_kernel<bf16_t><<<dim3(n, (int)blocks), 256, 0, (hipStream_t)stream>>>(p);
    else merge4_kernel<float><<<dim3(n, (int)blocks), 256, 0, (hipStream_t)stream>>>(p);
    return hipGetLastError();
}

}  // extern "C"
