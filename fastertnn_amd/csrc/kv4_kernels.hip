// A paged cache of keys and values in 4-bit codes: appending to it, reading it back, attention over it.  The layout is
// include/ftnn.h's (ftnn_kv4_t).
#include <algorithm>

#include "tokens_internal.h"

namespace ftnn {

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef unsigned int v4u __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

// a call's tokens and cache as the kernels use them
struct Kv4 {
    char* cache;
    const int32_t *table, *lens, *starts;
    int64_t pages, page_bytes, table_stride;
    int heads, dim, page, shift, sequences, tokens, width;   // page = 1 << shift
    int64_t head_bytes;

    // offsets in a block: key codes 0, value codes, keys' and values' (scale, zero)
    __device__ __forceinline__ int64_t values() const { return (int64_t)page * dim / 2; }
    __device__ __forceinline__ int64_t key_params() const { return (int64_t)page * dim; }
    __device__ __forceinline__ int64_t value_params() const { return (int64_t)page * (dim + 4); }
    // the page of position pos >= 0 of a sequence, or -1
    __device__ __forceinline__ int64_t page_of(int s, int64_t pos) const {
        const int64_t i = pos >> shift;
        if (i >= width) return -1;
        const int64_t id = table[s * table_stride + i];
        return id >= 0 && id < pages ? id : -1;
    }
    __device__ __forceinline__ char* block(int64_t id, int head) const { return cache + id * page_bytes + head * head_bytes; }
};
Kv4 device_view(const ftnn_kv4_t& k) {
    Kv4 v;
    v.cache = static_cast<char*>(k.d_cache), v.table = k.d_table, v.lens = k.d_lens, v.starts = k.d_starts;
    v.pages = k.pages, v.table_stride = k.table_stride, v.heads = k.heads, v.dim = k.dim, v.page = k.page;
    v.sequences = k.sequences, v.tokens = k.tokens, v.width = k.width;
    v.head_bytes = (int64_t)k.page * (k.dim + 8), v.page_bytes = v.head_bytes * k.heads;
    v.shift = 0;
    while ((1 << v.shift) < k.page) v.shift++;
    return v;
}

__device__ __forceinline__ int lane_id() { return threadIdx.x & 63; }

// the sequence of token row t, or -1 behind the last one: a wavefront compares 64 starts at a time
__device__ __forceinline__ int sequence_of(const Kv4& kv, int t) {
    int lo = 0, n = kv.sequences;
    while (n > 0) {
        const int stride = (n + 63) / 64, i = min((lane_id() + 1) * stride, n);
        const int c = __popcll(__ballot(lane_id() * stride < n && kv.starts[lo + i] <= t));
        lo += min(c * stride, n);
        n = min(stride, n - min(c * stride, n));
        if (stride == 1) break;
    }
    return lo < kv.sequences ? lo : -1;
}

// The tokens of a call that share a block of 8 positions, which the first of them stands for: count of them from row t on, or 0
// where t is not the first.  pos: of row t.
__device__ __forceinline__ int tokens_of_eight(const Kv4& kv, int t, int* s, int64_t* pos) {
    *s = sequence_of(kv, t);
    if (*s < 0) return 0;
    const int first = kv.starts[*s], end = min(kv.starts[*s + 1], kv.tokens);
    *pos = (int64_t)kv.lens[*s] - kv.starts[*s + 1] + t;
    if (t != first && (*pos & 7) != 0) return 0;
    return min(8 - (int)(*pos & 7), end - t);
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
    T e[8];
    __builtin_memcpy(e, p, sizeof(e));   // rows may start at any value
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = (float)e[i];
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; i++) e[i] = (T)x[i];
    __builtin_memcpy(p, e, sizeof(e));
}

// values d .. d + 7 of a row at position pos, rotated: products and sums in 64 bits, one rounding to fp32
template <typename T>
__device__ __forceinline__ void load_rotated(const T* row, int d, int64_t pos, const Kv4Rotation& r, float (&y)[8]) {
    float x[8];
    load8(row + d, x);
    const int half = r.rot / 2;
    const float *const c = r.cos + pos * half, *const n = r.sin + pos * half;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int e = d + i;
        if (e >= r.rot) {
            y[i] = x[i];
            continue;
        }
        const bool second = r.neighbours ? (e & 1) : e >= half;
        const int at = r.neighbours ? e / 2 : second ? e - half : e;
        const double other = r.neighbours ? (double)x[i ^ 1] : (double)(float)row[second ? e - half : e + half];
        const double a = (double)x[i] * (double)c[at], b = other * (double)n[at];   // exact
        y[i] = (float)(second ? a + b : a - b);
        asm volatile("" : "+v"(y[i]));   // in fp32 from here on: the compiler would make one rounding of this and a caller's to 16 bits
    }
}

// scale and zero of a group whose smallest and largest values are given, as the cache holds them: two bfloat16 in a word
__device__ __forceinline__ uint32_t make_params(float low, float high, bool fine, float* scale, float* zero) {
    const __bf16 z = (__bf16)low, s = (__bf16)(float)(((double)high - (double)low) / 15.0);
    *scale = (float)s, *zero = (float)z;
    if (!fine || !(__builtin_fabsf(*zero) < __builtin_inff())) {
        *scale = *zero = __builtin_nanf("");
        return 0x7FC07FC0u;
    }
    return (uint32_t)__builtin_bit_cast(unsigned short, s) | (uint32_t)__builtin_bit_cast(unsigned short, z) << 16;
}
__device__ __forceinline__ float scale_of(uint32_t params) { return __builtin_bit_cast(float, params << 16); }
__device__ __forceinline__ float zero_of(uint32_t params) { return __builtin_bit_cast(float, params & 0xFFFF0000u); }

// code of a value: in 64 bits, so that values next to a border come out as the formula says
__device__ __forceinline__ uint32_t code_of(float x, float scale, float zero) {
    if (!(scale > 0.0f)) return 0;
    const double q = __builtin_rint(((double)x - (double)zero) / (double)scale);
    return (uint32_t)__builtin_fmin(__builtin_fmax(q, 0.0), 15.0);
}

template <int LG>
__device__ __forceinline__ void group_range(const float (&y)[8], bool live, float* low, float* high, bool* fine) {
    float lo = __builtin_inff(), hi = -__builtin_inff();
    int ok = 1;
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (live) {
            lo = fminf(lo, y[i]), hi = fmaxf(hi, y[i]);
            ok &= __builtin_fabsf(y[i]) < __builtin_inff() ? 1 : 0;
        }
#pragma unroll
    for (int d = 1; d < LG; d *= 2) {
        lo = fminf(lo, __shfl_xor(lo, d)), hi = fmaxf(hi, __shfl_xor(hi, d));
        ok &= __shfl_xor(ok, d);
    }
    *low = lo, *high = hi, *fine = ok;
}

// One wavefront per (block of 8 positions, head): blockIdx.x is a token row, which works if it is the first of its block;
// blockIdx.y a head of keys and values, and behind those a head of queries.  The values of 8 tokens lie together, so the block has one
// owner, and a call's other tokens in it come through LDS.
template <typename T, int D>
__global__ __launch_bounds__(64) void k_kv4_append(Kv4 kv, Kv4Rows k, Kv4Rows v, Kv4Rotation r, int heads_q, Kv4Rows q, T* q_out) {
    constexpr int LG = D <= 64 ? 8 : D <= 128 ? 16 : 32, TPI = 64 / LG;   // lanes of a token, tokens at a time
    __shared__ __align__(8) uint8_t codes[8][D];
    const int t = blockIdx.x, lane = lane_id(), li = lane % LG, d = 8 * li;
    int s;
    int64_t pos;
    int count = tokens_of_eight(kv, t, &s, &pos);
    if (count <= 0 || pos < 0) return;
    if (r.rot && pos + count > r.positions) count = (int)max((int64_t)0, (int64_t)r.positions - pos);
    if (count <= 0) return;
    int head = blockIdx.y;
    if (head >= kv.heads) {
        head -= kv.heads;
        for (int i = lane / LG; i < count; i += TPI)
            if (d < D) {
                float y[8];
                load_rotated(static_cast<const T*>(q.p) + (t + i) * q.token_stride + head * q.head_stride, d, pos + i, r, y);
                store8(q_out + ((int64_t)(t + i) * heads_q + head) * D + d, y);
            }
        return;
    }
    const int64_t id = kv.page_of(s, pos);
    if (id < 0) return;
    char* const block = kv.block(id, head);
    const int slot = (int)(pos & (kv.page - 1));
    for (int i0 = 0; i0 < count; i0 += TPI) {
        const int i = i0 + lane / LG;
        const bool live = i < count && d < D;
#pragma unroll
        for (int which = 0; which < 2; which++) {
            float y[8] = {}, low, high, scale, zero;
            bool fine;
            if (live) {
                if (which == 0) load_rotated(static_cast<const T*>(k.p) + (t + i) * k.token_stride + head * k.head_stride, d, pos + i, r, y);
                else load8(static_cast<const T*>(v.p) + (t + i) * v.token_stride + head * v.head_stride + d, y);
            }
            group_range<LG>(y, live, &low, &high, &fine);
            const uint32_t params = make_params(low, high, fine, &scale, &zero);
            if (!live) continue;
            uint32_t w = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const uint32_t c = code_of(y[e], scale, zero);
                w |= c << (4 * e);
                if (which == 1) codes[i][d + e] = (uint8_t)c;
            }
            if (which == 0) *reinterpret_cast<uint32_t*>(block + (slot + i) * (D / 2) + d / 2) = w;
            if (li == 0) *reinterpret_cast<uint32_t*>(block + (which ? kv.value_params() : kv.key_params()) + (slot + i) * 4) = params;
        }
    }
    __syncthreads();
    uint32_t* const words = reinterpret_cast<uint32_t*>(block + kv.values()) + (slot / 8) * D;
    const int at = slot & 7;
    for (int e = lane; e < D; e += 64) {
        uint32_t w = 0;
        for (int i = 0; i < count; i++) w |= (uint32_t)codes[i][e] << (4 * (at + i));
        if (count < 8) w |= words[e] & ~((0xFFFFFFFFu >> (32 - 4 * count)) << (4 * at));
        words[e] = w;
    }
}

template <typename T, int D>
__global__ __launch_bounds__(64) void k_kv4_read(Kv4 kv, T* K, T* V) {
    constexpr int LG = D <= 64 ? 8 : D <= 128 ? 16 : 32, TPI = 64 / LG;
    const int t = blockIdx.x, head = blockIdx.y, lane = lane_id(), d = 8 * (lane % LG);
    int s;
    int64_t pos;
    const int count = tokens_of_eight(kv, t, &s, &pos);
    if (count <= 0) return;
    const int64_t id = pos >= 0 ? kv.page_of(s, pos) : -1;
    const char* const block = kv.block(max(id, (int64_t)0), head);
    const int slot = (int)(pos & (kv.page - 1));
    if (K)
        for (int i = lane / LG; i < count; i += TPI)
            if (d < D) {
                float y[8] = {};
                if (id >= 0) {
                    const uint32_t w = *reinterpret_cast<const uint32_t*>(block + (slot + i) * (D / 2) + d / 2);
                    const uint32_t p = *reinterpret_cast<const uint32_t*>(block + kv.key_params() + (slot + i) * 4);
#pragma unroll
                    for (int e = 0; e < 8; e++) y[e] = __builtin_fmaf((float)(w >> (4 * e) & 15u), scale_of(p), zero_of(p));
                }
                store8(K + ((int64_t)(t + i) * kv.heads + head) * D + d, y);
            }
    if (V) {
        const uint32_t* const words = reinterpret_cast<const uint32_t*>(block + kv.values()) + (slot / 8) * D;
        for (int e = lane; e < D; e += 64) {
            const uint32_t w = id >= 0 ? words[e] : 0u;
            for (int i = 0; i < count; i++) {
                const uint32_t p = id >= 0 ? *reinterpret_cast<const uint32_t*>(block + kv.value_params() + (slot + i) * 4) : 0u;
                V[((int64_t)(t + i) * kv.heads + head) * D + e] = (T)__builtin_fmaf((float)(w >> (4 * ((slot + i) & 7)) & 15u), scale_of(p), zero_of(p));
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------------------- attention
//
// Scores and outputs come from v_mfma_f32_16x16x32_bf16 on the codes themselves: 128 + code is a bfloat16 whose lowest mantissa bits
// are the code, so two codes become an operand word with an AND and an OR, and a scale and a zero per token make
//     q . k_t = ks_t (sum_d q_d (128 + c_td) - 128 sum_d q_d) + kz_t sum_d q_d
//     sum_t p_t v_td = sum_t w_t (128 + c_td) - 136 sum_t w_t + sum_t p_t (vz_t + 8 vs_t),   w_t = p_t vs_t
// with w_t rounded to bfloat16 (of FTNN_F16: the sum of two) in both of its sums, so that its rounding only meets code - 8, which is
// what is rounded where values are multiplied.  The cancelled 128 costs 2^-24 * 128 of a code, far below that.
//
// A step is 32 tokens of one wavefront.  Keys are the A operand: row r of block b (two blocks of 16) is token 8 (r / 4) + 4 b + r % 4, so that
// lane quarter g ends with the scores of tokens 8 g .. 8 g + 7 of its column (a query), in the order in which the second product takes
// its weights as B operand: no lanes are exchanged.  The values of 8 tokens of a channel are one word of the cache, its A operand.
// Rows of a tile are (token, query head of the group) pairs of one sequence and one head of keys.

__device__ __forceinline__ v8bf codes8(uint32_t w) {
    v4u r;
#pragma unroll
    for (int p = 0; p < 4; p++) r[p] = (w >> (4 * p) & 0x000F000Fu) | 0x43004300u;
    return __builtin_bit_cast(v8bf, r);
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    return (uint32_t)__builtin_bit_cast(unsigned short, (__bf16)a) | (uint32_t)__builtin_bit_cast(unsigned short, (__bf16)b) << 16;
}
__device__ __forceinline__ float bf16_low(uint32_t w) { return __builtin_bit_cast(float, w << 16); }
__device__ __forceinline__ float bf16_high(uint32_t w) { return __builtin_bit_cast(float, w & 0xFFFF0000u); }

// eight values as operand words: word p holds elements p and p + 4, as codes8 has them; the rest in `low` where PARTS is 2
template <int PARTS>
__device__ __forceinline__ void split8(const float (&x)[8], v8bf& high, v8bf& low) {
    v4u h, l;
#pragma unroll
    for (int p = 0; p < 4; p++) {
        h[p] = pack_bf16(x[p], x[p + 4]);
        if (PARTS == 2) l[p] = pack_bf16(x[p] - bf16_low(h[p]), x[p + 4] - bf16_high(h[p]));
    }
    high = __builtin_bit_cast(v8bf, h);
    if (PARTS == 2) low = __builtin_bit_cast(v8bf, l);
}

struct Kv4Attend {
    Kv4 kv;
    Kv4Rows q;
    int heads_q, group, splits;
    float scale2;      // scale * log2(e)
    void* out;
    float* part;       // [splits][tokens * heads_q][dim], then [splits][tokens * heads_q][2]: sums, maximum and sum of weights
};

constexpr int kTile = 16;   // rows of a tile

// which tile of which sequence a workgroup's number is; false behind the last
__device__ __forceinline__ bool find_tile(const Kv4& kv, int group, int number, int* s, int* tile) {
    int before = 0;
    for (int b0 = 0; b0 < kv.sequences; b0 += 64) {
        const int b = b0 + lane_id();
        int64_t rows = 0;
        if (b < kv.sequences) rows = (int64_t)max(0, min(kv.starts[b + 1], kv.tokens) - max(kv.starts[b], 0)) * group;
        const int tiles = (int)((rows + kTile - 1) / kTile);
        int sum = tiles;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int o = __shfl_up(sum, d);
            if (lane_id() >= d) sum += o;
        }
        const uint64_t past = __ballot(before + sum > number);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            *s = b0 + l;
            *tile = number - before - (__shfl(sum, l) - __shfl(tiles, l));
            return true;
        }
        before += __shfl(sum, 63);
    }
    return false;
}

template <typename T, int D>
__global__ __launch_bounds__(256) void k_kv4_attend(Kv4Attend p) {
    constexpr int PARTS = std::is_same<T, _Float16>::value ? 2 : 1, ND = D / 32, NB = D / 16, WAVES = 4;
    extern __shared__ float lds[];   // [WAVES][16][D + 4] sums, then [WAVES][16][2]
    const Kv4& kv = p.kv;
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    int s, tile;
    if (!find_tile(kv, p.group, blockIdx.x, &s, &tile)) return;
    s = __builtin_amdgcn_readfirstlane(s), tile = __builtin_amdgcn_readfirstlane(tile);
    const int head = blockIdx.y, split = blockIdx.z;
    const int first = max(kv.starts[s], 0), end = min(kv.starts[s + 1], kv.tokens), n = end - first;
    const int64_t held = min((int64_t)max(kv.lens[s], 0), (int64_t)kv.width << kv.shift);
    // row: token j of the call's n, query head of the group
    const int64_t row = (int64_t)tile * kTile + c, rows = (int64_t)n * p.group;
    const bool live = row < rows;
    const int j = live ? (int)(row / p.group) : n - 1, hq = head * p.group + (live ? (int)(row % p.group) : 0);
    const int64_t base = (int64_t)kv.lens[s] - kv.starts[s + 1] + first;   // position of token 0
    const int64_t seen = max((int64_t)0, min(held, base + j + 1));         // tokens that the row sees
    const int64_t last_row = min((int64_t)tile * kTile + kTile, rows) - 1;
    const int64_t most = max((int64_t)0, min(held, base + last_row / p.group + 1)), least = max((int64_t)0, min(held, base + (int64_t)tile * kTile / p.group + 1));
    // queries: word j of a lane's D / 4 channels 8 words apart per quarter
    v8bf qh[ND], ql[PARTS == 2 ? ND : 1];
    float qsum = 0.0f;
    const T* const q = static_cast<const T*>(p.q.p) + (int64_t)(first + j) * p.q.token_stride + (int64_t)hq * p.q.head_stride + g * (D / 4);
#pragma unroll
    for (int i = 0; i < ND; i++) {
        float x[8];
        load8(q + 8 * i, x);
#pragma unroll
        for (int e = 0; e < 8; e++) qsum += x[e];
        split8<PARTS>(x, qh[i], ql[PARTS == 2 ? i : 0]);
    }
    qsum += __shfl_xor(qsum, 16);
    qsum += __shfl_xor(qsum, 32);
    v4f o[NB], wsum = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < NB; i++) o[i] = v4f{0, 0, 0, 0};
    float m = -__builtin_inff(), l = 0.0f, zsum = 0.0f;
    const v4u ones_w = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
    const v8bf ones = __builtin_bit_cast(v8bf, ones_w);

    const int64_t steps = (most + 31) / 32, per = (steps + p.splits - 1) / p.splits, from = per * split, to = min(steps, from + per);
    for (int64_t st = from + wave; st < to; st += WAVES) {
        const int64_t t0 = st * 32;
        // keys: this lane's row of each block; (scale, zero) and values: tokens 8 g .. 8 g + 7
        uint32_t kw[2][ND], vw[NB], kp[8], vp[8];
        bool there;
        {
            const int64_t kt = t0 + 8 * (c >> 2) + (c & 3);   // + 4 b
            const int64_t id = kv.page_of(s, kt);
            const char* const b = kv.block(max(id, (int64_t)0), head) + (kt & (kv.page - 1)) * (D / 2) + g * (D / 8);
            __builtin_memcpy(kw[0], __builtin_assume_aligned(b, 4), 4 * ND);
            __builtin_memcpy(kw[1], __builtin_assume_aligned(b + 4 * (D / 2), 4), 4 * ND);
        }
        {
            const int64_t vt = t0 + 8 * g, id = kv.page_of(s, vt), slot = vt & (kv.page - 1);
            there = id >= 0;
            const char* const b = kv.block(max(id, (int64_t)0), head);
            __builtin_memcpy(vw, __builtin_assume_aligned(b + kv.values() + ((slot / 8) * D + c * NB) * 4, 8), 4 * NB);
            __builtin_memcpy(kp, __builtin_assume_aligned(b + kv.key_params() + slot * 4, 16), 32);
            __builtin_memcpy(vp, __builtin_assume_aligned(b + kv.value_params() + slot * 4, 16), 32);
        }
        float sc[8];
#pragma unroll
        for (int b = 0; b < 2; b++) {
            v4f a = {-128.0f * qsum, -128.0f * qsum, -128.0f * qsum, -128.0f * qsum};
#pragma unroll
            for (int i = 0; i < ND; i++) {
                const v8bf k = codes8(kw[b][i]);
                a = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, qh[i], a, 0, 0, 0);
                if (PARTS == 2) a = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, ql[i], a, 0, 0, 0);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) sc[4 * b + e] = __builtin_fmaf(a[e], scale_of(kp[4 * b + e]), qsum * zero_of(kp[4 * b + e]));
        }
        if (t0 + 32 > least || !__all(there)) {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (!there || t0 + 8 * g + e >= seen) sc[e] = -__builtin_inff(), vp[e] = 0u;   // what lies there is not looked at
        }
        float top = m;
#pragma unroll
        for (int e = 0; e < 8; e++) top = fmaxf(top, sc[e]);
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float safe = top == -__builtin_inff() ? 0.0f : top;
        if (__any(top > m)) {
            const float f = __builtin_amdgcn_exp2f((m - safe) * p.scale2);
            l *= f, zsum *= f, wsum *= f;
#pragma unroll
            for (int i = 0; i < NB; i++) o[i] *= f;
            m = top;
        }
        float w[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float x = __builtin_amdgcn_exp2f((sc[e] - safe) * p.scale2);
            l += x;
            zsum = __builtin_fmaf(x, __builtin_fmaf(8.0f, scale_of(vp[e]), zero_of(vp[e])), zsum);
            w[e] = x * scale_of(vp[e]);
        }
        v8bf wh, wl;
        split8<PARTS>(w, wh, wl);
        wsum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, wh, wsum, 0, 0, 0);
        if (PARTS == 2) wsum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, wl, wsum, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < NB; i++) {
            const v8bf a = codes8(vw[i]);
            o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, wh, o[i], 0, 0, 0);
            if (PARTS == 2) o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, wl, o[i], 0, 0, 0);
        }
    }
    l += __shfl_xor(l, 16), zsum += __shfl_xor(zsum, 16);
    l += __shfl_xor(l, 32), zsum += __shfl_xor(zsum, 32);
    // the wavefronts meet: sums of a row, channel (4 g + e) NB + i of block i in accumulator e
    constexpr int LD = D + 4;
    float* const mine = lds + (wave * 16 + c) * LD;
#pragma unroll
    for (int i = 0; i < NB; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) mine[(4 * g + e) * NB + i] = o[i][e] - 136.0f * wsum[e] + zsum;
    float* const ml = lds + WAVES * 16 * LD;
    if (g == 0) ml[(wave * 16 + c) * 2] = m, ml[(wave * 16 + c) * 2 + 1] = l;
    __syncthreads();
    for (int x = threadIdx.x; x < 16 * D; x += 256) {
        const int r = x / D, d = x % D;
        const int64_t rr = (int64_t)tile * kTile + r;
        if (rr >= rows) break;
        float top = -__builtin_inff(), sum = 0.0f, den = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; w++) top = fmaxf(top, ml[(w * 16 + r) * 2]);
        const float safe = top == -__builtin_inff() ? 0.0f : top;
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            const float f = __builtin_amdgcn_exp2f((ml[(w * 16 + r) * 2] - safe) * p.scale2);
            sum = __builtin_fmaf(lds[(w * 16 + r) * LD + d], f, sum);
            den = __builtin_fmaf(ml[(w * 16 + r) * 2 + 1], f, den);
        }
        const int64_t at = (int64_t)(first + rr / p.group) * p.heads_q + head * p.group + rr % p.group;
        if (p.splits == 1) {
            static_cast<T*>(p.out)[at * D + d] = (T)(den == 0.0f ? 0.0f : sum / den);
        } else {
            const int64_t all = (int64_t)kv.tokens * p.heads_q;
            p.part[(split * all + at) * D + d] = sum;
            if (d == 0) {
                float* const pm = p.part + p.splits * all * D + (split * all + at) * 2;
                pm[0] = top, pm[1] = den;
            }
        }
    }
}

// the parts of a row meet
template <typename T, int D>
__global__ __launch_bounds__(64) void k_kv4_join(Kv4Attend p) {
    const int64_t all = (int64_t)p.kv.tokens * p.heads_q, at = blockIdx.x;
    const int token = (int)(at / p.heads_q);
    if (token < p.kv.starts[0] || token >= p.kv.starts[p.kv.sequences]) return;
    const float* const pm = p.part + p.splits * all * D;
    float top = -__builtin_inff(), den = 0.0f, sum[(D + 63) / 64] = {};
    for (int i = 0; i < p.splits; i++) top = fmaxf(top, pm[(i * all + at) * 2]);
    const float safe = top == -__builtin_inff() ? 0.0f : top;
    for (int i = 0; i < p.splits; i++) {
        const float f = __builtin_amdgcn_exp2f((pm[(i * all + at) * 2] - safe) * p.scale2);
        den = __builtin_fmaf(pm[(i * all + at) * 2 + 1], f, den);
#pragma unroll
        for (int x = 0; x < (D + 63) / 64; x++)
            if (x * 64 + lane_id() < D) sum[x] = __builtin_fmaf(p.part[(i * all + at) * D + x * 64 + lane_id()], f, sum[x]);
    }
#pragma unroll
    for (int x = 0; x < (D + 63) / 64; x++)
        if (x * 64 + lane_id() < D) static_cast<T*>(p.out)[at * D + x * 64 + lane_id()] = (T)(den == 0.0f ? 0.0f : sum[x] / den);
}

// fn(the head size as a constant)
template <typename F>
hipError_t with_dim(int dim, F&& fn) {
    switch (dim) {
        case 64: return fn(std::integral_constant<int, 64>{});
        case 96: return fn(std::integral_constant<int, 96>{});
        case 128: return fn(std::integral_constant<int, 128>{});
        default: return fn(std::integral_constant<int, 256>{});
    }
}

int64_t tiles_of(const ftnn_kv4_t& kv, int group) {   // at most: tokens of a sequence share tiles, sequences do not
    const int64_t t = kv.tokens;
    return std::min((t * group + kTile - 1) / kTile + kv.sequences, t * ((group + kTile - 1) / kTile));
}

int splits_of(const ftnn_kv4_t& kv, int heads_q, int max_len) {
    const int64_t most = max_len > 0 ? std::min<int64_t>(max_len, (int64_t)kv.width * kv.page) : (int64_t)kv.width * kv.page;
    const int64_t base = std::max<int64_t>(1, tiles_of(kv, heads_q / kv.heads) * kv.heads);
    return (int)std::max<int64_t>(1, std::min<int64_t>({512 / base, (most + 255) / 256, 64}));
}

}  // namespace

hipError_t launch_kv4_append(const ftnn_kv4_t& kv, int dtype, const Kv4Rows& k, const Kv4Rows& v, const Kv4Rotation& r, int heads_q,
                             const Kv4Rows& q, void* d_q_out, hipStream_t st) {
    const Kv4 dv = device_view(kv);
    return with_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        return with_dim(kv.dim, [&](auto d) {
            k_kv4_append<T, decltype(d)::value><<<dim3(kv.tokens, kv.heads + heads_q), dim3(64), 0, st>>>(dv, k, v, r, heads_q, q, static_cast<T*>(d_q_out));
            return hipGetLastError();
        });
    });
}

hipError_t launch_kv4_read(const ftnn_kv4_t& kv, int dtype, void* d_k, void* d_v, hipStream_t st) {
    const Kv4 dv = device_view(kv);
    return with_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        return with_dim(kv.dim, [&](auto d) {
            k_kv4_read<T, decltype(d)::value><<<dim3(kv.tokens, kv.heads), dim3(64), 0, st>>>(dv, static_cast<T*>(d_k), static_cast<T*>(d_v));
            return hipGetLastError();
        });
    });
}

int64_t kv4_attention_scratch(const ftnn_kv4_t& kv, int heads_q, int max_len) {
    const int64_t splits = splits_of(kv, heads_q, max_len);
    return splits == 1 ? 0 : splits * kv.tokens * heads_q * (kv.dim + 2) * 4;
}

hipError_t launch_kv4_attention(const ftnn_kv4_t& kv, int dtype, int heads_q, const Kv4Rows& q, float scale, int max_len, void* d_out,
                                void* d_scratch, hipStream_t st) {
    Kv4Attend p;
    p.kv = device_view(kv), p.q = q, p.heads_q = heads_q, p.group = heads_q / kv.heads, p.splits = splits_of(kv, heads_q, max_len);
    p.scale2 = scale * 1.44269504088896341f, p.out = d_out, p.part = static_cast<float*>(d_scratch);
    const int64_t tiles = tiles_of(kv, p.group);
    auto go = [&](auto t) {
        typedef decltype(t) T;
        return with_dim(kv.dim, [&](auto d) {
            constexpr int D = decltype(d)::value;
            const size_t bytes = 4 * 16 * (D + 4 + 2) * 4;
            static const hipError_t set = hipFuncSetAttribute(reinterpret_cast<const void*>(k_kv4_attend<T, D>), hipFuncAttributeMaxDynamicSharedMemorySize, 160 << 10);
            if (set != hipSuccess) return set;
            k_kv4_attend<T, D><<<dim3((unsigned)tiles, kv.heads, p.splits), dim3(256), bytes, st>>>(p);
            hipError_t e = hipGetLastError();
            if (e != hipSuccess || p.splits == 1) return e;
            k_kv4_join<T, D><<<dim3((unsigned)((int64_t)kv.tokens * heads_q)), dim3(64), 0, st>>>(p);
            return hipGetLastError();
        });
    };
    return dtype == FTNN_F16 ? go((_Float16)0.0f) : go((__bf16)0.0f);
}

}  // namespace ftnn
