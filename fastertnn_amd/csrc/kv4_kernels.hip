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

// The tokens of a call that share a block of 8 positions: their rows t .. t + count - 1 of sequence s, from position pos on.  The values of a block lie in
// the same words, so it has one owner: number `number` of the call's blocks, counted sequence by sequence.  count is 0 behind the last.
struct Kv4Eight {
    int s, t, count, pos;
};
__device__ __forceinline__ Kv4Eight find_eight(const Kv4& kv, int number) {
    int before = 0;
    for (int b0 = 0; b0 < kv.sequences; b0 += 64) {
        const int b = min(b0 + lane_id(), kv.sequences - 1);
        const int from = kv.starts[b], to = kv.starts[b + 1], length = kv.lens[b], first = max(from, 0), end = min(to, kv.tokens);   // together: one wait
        // position of row `first`; negative where a sequence has more new tokens than it holds: its blocks are counted too
        const int pos = max(length, 0) - to + first, rows = b0 + lane_id() < kv.sequences ? end - first : 0;
        const int blocks = rows > 0 ? ((pos + rows - 1) >> 3) - (pos >> 3) + 1 : 0;
        int sum = blocks;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int o = __shfl_up(sum, d);
            if (lane_id() >= d) sum += o;
        }
        const uint64_t past = __ballot(before + sum > number);
        if (past) {
            const int l = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)past) - 1);
            auto at = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
            const int row0 = at(first), n = at(rows), p0 = at(pos), i = number - before - at(sum) + at(blocks), done = i == 0 ? 0 : 8 * i - (p0 & 7);
            return {b0 + l, row0 + done, min(8 - ((p0 + done) & 7), n - done), p0 + done};
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    return {0, 0, 0, 0};
}
// blocks of 8 positions at most: a sequence's first and last may be cut
int eights_of(const ftnn_kv4_t& kv) { return (int)std::min<int64_t>(kv.tokens, ((int64_t)kv.tokens + 7) / 8 + 2 * (int64_t)kv.sequences); }

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
    T e[8];
    __builtin_memcpy(e, p, sizeof(e));   // rows may start at any value
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = (float)e[i];
}
// the same in two steps: as they lie, and as numbers
template <typename T>
struct Eight {
    uint32_t w[2 * sizeof(T)];
    __device__ __forceinline__ void load(const T* p) { __builtin_memcpy(w, p, sizeof(w)); }
    __device__ __forceinline__ void numbers(float (&x)[8]) const {
        T e[8];
        __builtin_memcpy(e, w, sizeof(w));
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = (float)e[i];
    }
};
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; i++) e[i] = (T)x[i];
    __builtin_memcpy(p, e, sizeof(e));
}

// cosines and sines of elements d .. d + 7 at a position, the sines with the sign of their term; what is not rotated has none
struct Kv4Angles {
    float c[8], n[8];
};
__device__ __forceinline__ void load_angles(const Kv4Rotation& r, int pos, int d, Kv4Angles& a) {
    if (d >= r.rot) return;
    const int half = r.rot / 2;
    const float *const c = r.cos + (int64_t)pos * half, *const n = r.sin + (int64_t)pos * half;
    if (r.neighbours && d + 8 <= r.rot) {   // whole pairs: four entries
        float c4[4], n4[4];
        __builtin_memcpy(c4, c + d / 2, 16), __builtin_memcpy(n4, n + d / 2, 16);
#pragma unroll
        for (int i = 0; i < 8; i++) a.c[i] = c4[i / 2], a.n[i] = n4[i / 2];
    } else if (!r.neighbours && half % 8 == 0) {   // all of one half
        const int at = d >= half ? d - half : d;
        __builtin_memcpy(a.c, c + at, 32), __builtin_memcpy(a.n, n + at, 32);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int e = min(d + i, r.rot - 1), at = r.neighbours ? e / 2 : e >= half ? e - half : e;   // (what is behind stays as it is)
            a.c[i] = c[at], a.n[i] = n[at];
        }
    }
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (!(r.neighbours ? (i & 1) : d + i >= half)) a.n[i] = -a.n[i];
}
// values d .. d + 7 of a row and, where they are rotated, the other elements of their pairs
template <typename T>
__device__ __forceinline__ void load_pairs(const T* row, int d, const Kv4Rotation& r, Eight<T>& x, Eight<T>& other) {
    x.load(row + d);
    if (d >= r.rot || r.neighbours) return;   // (neighbours are among the eight)
    const int half = r.rot / 2;
    if (half % 8 == 0) {
        other.load(row + (d >= half ? d - half : d + half));
    } else {
        T e[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int at = min(d + i, r.rot - 1);
            e[i] = row[at >= half ? at - half : at + half];
        }
        __builtin_memcpy(other.w, e, sizeof(e));
    }
}
// rotated: products and sums in 64 bits, one rounding to fp32
__device__ __forceinline__ void rotate(const Kv4Rotation& r, int d, const Kv4Angles& a, float (&x)[8], const float (&other)[8]) {
    if (d >= r.rot) return;
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const double q = (double)(r.neighbours ? x[i ^ 1] : other[i]) * (double)a.n[i];   // exact, as is the other product
        y[i] = (float)__builtin_fma((double)x[i], (double)a.c[i], q);
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        if (d + i < r.rot) x[i] = y[i];
        asm volatile("" : "+v"(x[i]));   // in fp32 from here on: the compiler would make one rounding of this and a caller's to 16 bits
    }
}

// scale and zero of a group whose smallest and largest values are given, as the cache holds them: two bfloat16 in a word
__device__ __forceinline__ uint32_t make_params(float low, float high, float* scale, float* zero) {
    float fifteenth = (float)(((double)high - (double)low) * (1.0 / 15.0));   // (times 1/15 in 64 bits: one rounding to fp32 is the quotient's)
    asm volatile("" : "+v"(fifteenth));   // in fp32 from here on: the compiler would make one rounding of this and the next
    const __bf16 z = (__bf16)low, s = (__bf16)fifteenth;
    *scale = (float)s, *zero = (float)z;
    if (!(__builtin_fabsf(*zero) < __builtin_inff())) {   // of a group with a NaN or an infinity, or a zero beyond bfloat16
        *scale = *zero = __builtin_nanf("");
        return 0x7FC07FC0u;
    }
    return (uint32_t)__builtin_bit_cast(unsigned short, s) | (uint32_t)__builtin_bit_cast(unsigned short, z) << 16;
}
__device__ __forceinline__ float scale_of(uint32_t params) { return __builtin_bit_cast(float, params << 16); }
__device__ __forceinline__ float zero_of(uint32_t params) { return __builtin_bit_cast(float, params & 0xFFFF0000u); }

// Eight codes.  A difference, the reciprocal and a product in fp32 are off by at most (2^-24 + 2^-23 + 2^-24) of a quotient of up to 16, 2^-18: where none of
// the eight is within 2^-16 of a border between codes they are what the formula says.  Others are divided in 64 bits.  Adding 1.5 * 2^23 rounds to a whole
// number, ties to even, which is the lowest bits of the sum; the bits of the constant, moved along, are taken off at the end.
__device__ __forceinline__ uint32_t codes_of(const float (&x)[8], float scale, float zero, float high) {
    if (!(scale > 0.0f)) return 0;
    constexpr uint32_t kBits = 0x4B400000u;
    constexpr uint32_t kOnes = 0x11111111u;   // sum of 16^e
    const float inv = __builtin_amdgcn_rcpf(scale);
    uint32_t w = 0;
    float far = 0.0f;   // the largest distance from a whole number
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float q = __builtin_amdgcn_fmed3f((x[e] - zero) * inv, 0.0f, 15.0f), t = q + 12582912.0f;
        far = fmaxf(far, __builtin_fabsf(q - (t - 12582912.0f)));
        w += __builtin_bit_cast(uint32_t, t) << (4 * e);
    }
    w -= kBits * kOnes;
    if (far > 0.5f - 0x1p-16f || scale < 0x1p-100f || !(high - zero < __builtin_inff())) {   // (a difference beyond fp32, a scale without a reciprocal)
        w = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const double q = __builtin_rint(((double)x[e] - (double)zero) / (double)scale);
            w |= (uint32_t)__builtin_fmin(__builtin_fmax(q, 0.0), 15.0) << (4 * e);
        }
    }
    return w;
}

// lane i and the lane that differs from it in bit B alone, once all lower bits agree: exchanged in the vector ALU
template <int B>
__device__ __forceinline__ float across(float x) {
    const int v = __builtin_bit_cast(int, x);
    if constexpr (B == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
        return __builtin_bit_cast(float, (uint32_t)((lane_id() & 16) ? r[0] : r[1]));
    } else {
        // quad_perm [1,0,3,2], quad_perm [2,3,0,1], row_half_mirror, row_mirror
        constexpr int ctrl = B == 1 ? 0xB1 : B == 2 ? 0x4E : B == 4 ? 0x141 : 0x140;
        return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, v, ctrl, 0xF, 0xF, false));
    }
}

// smallest and largest value of the LG lanes that hold a token; of one with a NaN or an infinity the smallest is -infinity
template <int LG>
__device__ __forceinline__ void group_range(const float (&y)[8], bool live, float* low, float* high) {
    float lo = __builtin_inff(), hi = -__builtin_inff();
    if (live) {
        float none = 0.0f;   // 0 times a NaN or an infinity is a NaN
        lo = hi = y[0];
#pragma unroll
        for (int i = 1; i < 8; i++) lo = fminf(lo, y[i]), hi = fmaxf(hi, y[i]);
#pragma unroll
        for (int i = 0; i < 8; i++) none = __builtin_fmaf(y[i], 0.0f, none);
        lo = none == 0.0f ? lo : -__builtin_inff();
    }
    auto step = [&](float l, float h) { lo = fminf(lo, l), hi = fmaxf(hi, h); };
    step(across<1>(lo), across<1>(hi));
    step(across<2>(lo), across<2>(hi));
    step(across<4>(lo), across<4>(hi));
    if constexpr (LG > 8) step(across<8>(lo), across<8>(hi));
    if constexpr (LG > 16) step(across<16>(lo), across<16>(hi));
    *low = lo, *high = hi;
}

// A wavefront per (block of 8 positions, head of keys and values, or behind those of queries); where there are many it takes one head after the other, so
// that finding the block is paid once for several.  Of many tokens the vector ALU bounds it, with the angles' 64-bit products and the codes (busy 76 % of the
// launch): 5 x 4001 new tokens, 8 heads of 64 with 16 of queries: 35 us for 108 MB (3.1 TB/s).  Of few it is the chain of loads (starts, table, rows): 48 x 1
// of 8 + 32 heads of 128: 7 us on the device, where an empty launch is 2.4.  LG lanes hold a token's channels, eight each.  The codes of a block's values meet in LDS, where every lane makes the words of its channels; what the block holds already of
// other tokens stays.
template <typename T, int D>
__global__ __launch_bounds__(256) void k_kv4_append(Kv4 kv, Kv4Rows k, Kv4Rows v, Kv4Rotation r, int heads_q, Kv4Rows q, T* q_out) {
    constexpr int LG = D <= 64 ? 8 : D <= 128 ? 16 : 32, TPI = 64 / LG;   // lanes of a token, tokens at a time
    __shared__ uint32_t codes[4][8][D / 8];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane % LG, d = 8 * li;
    const Kv4Eight at = find_eight(kv, blockIdx.x);
    const int count = r.rot ? min(at.count, r.positions - at.pos) : at.count;
    if (count <= 0 || at.pos < 0) return;
    const int64_t id = kv.page_of(at.s, at.pos);
    const int slot = at.pos & (kv.page - 1), place = slot & 7;
    constexpr int JS = 8 / TPI;
    Kv4Angles angles[JS];   // of the lane's channels: the same for all heads
#pragma unroll
    for (int j = 0; j < JS; j++) {
        const int i = j * TPI + lane / LG;
        if (i < count && d < D) load_angles(r, at.pos + i, d, angles[j]);
    }
    // a head's rows of the block, all asked for at once
    struct Rows {
        Eight<T> x[JS], other[JS], value[JS];
    };
    const int heads = kv.heads + heads_q, step = 4 * gridDim.y;
    auto fetch = [&](int head, Rows& rows) {
        const bool query = head >= kv.heads;
        const T* const from = query ? static_cast<const T*>(q.p) + at.t * q.token_stride + (head - kv.heads) * q.head_stride
                                    : static_cast<const T*>(k.p) + at.t * k.token_stride + head * k.head_stride;
        const T* const values = static_cast<const T*>(v.p) + at.t * v.token_stride + head * v.head_stride;
        const int64_t stride = query ? q.token_stride : k.token_stride;
#pragma unroll
        for (int j = 0; j < JS; j++) {
            const int i = j * TPI + lane / LG;
            if (i < count && d < D) {
                load_pairs(from + i * stride, d, r, rows.x[j], rows.other[j]);
                if (!query) rows.value[j].load(values + i * v.token_stride + d);
            }
        }
    };
    for (int head = blockIdx.y * 4 + wave; head < heads; head += step) {   // (no wavefront waits for another)
        Rows rows;
        fetch(head, rows);
#pragma unroll
        for (int j = 0; j < JS; j++)
#pragma unroll
            for (int e = 0; e < 8; e++) asm volatile("" : "+v"(angles[j].c[e]), "+v"(angles[j].n[e]));   // (kept in 32 bits between heads)
        const bool query = head >= kv.heads;
        if (!query && id < 0) continue;
        float y[JS][8];
#pragma unroll
        for (int j = 0; j < JS; j++) {
            float other[8];
            rows.x[j].numbers(y[j]), rows.other[j].numbers(other);
            rotate(r, d, angles[j], y[j], other);
        }
        if (query) {
#pragma unroll
            for (int j = 0; j < JS; j++) {
                const int i = j * TPI + lane / LG;
                if (i < count && d < D) store8(q_out + ((int64_t)(at.t + i) * heads_q + head - kv.heads) * D + d, y[j]);
            }
            continue;
        }
        char* const block = kv.block(id, head);
#pragma unroll
        for (int which = 0; which < 2; which++) {
#pragma unroll
            for (int j = 0; j < JS; j++)
                if (which == 1) rows.value[j].numbers(y[j]);
#pragma unroll
            for (int j = 0; j < JS; j++) {
                if (j * TPI >= count) break;
                const int i = j * TPI + lane / LG;
                const bool live = i < count && d < D;
                float low, high, scale, zero;
                group_range<LG>(y[j], live, &low, &high);
                const uint32_t params = make_params(low, high, &scale, &zero);
                if (live) {
                    const uint32_t w = codes_of(y[j], scale, zero, high);
                    if (which == 0) *reinterpret_cast<uint32_t*>(block + (slot + i) * (D / 2) + d / 2) = w;
                    else codes[wave][i][li] = w;
                    if (li == 0) *reinterpret_cast<uint32_t*>(block + (which ? kv.value_params() : kv.key_params()) + (slot + i) * 4) = params;
                }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");   // the wavefront's own codes: its LDS accesses keep their order
        __builtin_amdgcn_wave_barrier();
        uint32_t* const words = reinterpret_cast<uint32_t*>(block + kv.values()) + (slot / 8) * D;
        for (int e = lane; e < D; e += 64) {
            uint32_t w = 0;
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (i < count) w |= (codes[wave][i][e / 8] >> (4 * (e & 7)) & 15u) << (4 * (place + i));
            if (count < 8) w |= words[e] & ~((0xFFFFFFFFu >> (32 - 4 * count)) << (4 * place));
            words[e] = w;
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// The same blocks and lanes the other way round: a lane's eight channels of a token are one word of keys, and eight words that hold its token among others,
// which the block's other lanes find in the L1.  Stores bound it: the tokens above in 11 us, 33 MB of results.
template <typename T, int D>
__global__ __launch_bounds__(256) void k_kv4_read(Kv4 kv, T* K, T* V) {
    constexpr int LG = D <= 64 ? 8 : D <= 128 ? 16 : 32, TPI = 64 / LG;
    const int lane = lane_id(), head = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), d = 8 * (lane % LG);
    if (head >= kv.heads) return;
    const Kv4Eight at = find_eight(kv, blockIdx.x);
    if (at.count <= 0) return;
    const int64_t id = at.pos >= 0 ? kv.page_of(at.s, at.pos) : -1;
    const char* const block = kv.block(max(id, (int64_t)0), head);
    const int slot = at.pos & (kv.page - 1);
    const uint32_t* const words = reinterpret_cast<const uint32_t*>(block + kv.values()) + (slot / 8) * D + d;
#pragma unroll
    for (int i0 = 0; i0 < 8; i0 += TPI) {
        const int i = i0 + lane / LG;
        if (i >= at.count || d >= D) continue;
        const int64_t to = ((int64_t)(at.t + i) * kv.heads + head) * D + d;
        if (K) {
            float y[8] = {};
            if (id >= 0) {
                const uint32_t w = *reinterpret_cast<const uint32_t*>(block + (slot + i) * (D / 2) + d / 2);
                const uint32_t p = *reinterpret_cast<const uint32_t*>(block + kv.key_params() + (slot + i) * 4);
#pragma unroll
                for (int e = 0; e < 8; e++) y[e] = __builtin_fmaf((float)(w >> (4 * e) & 15u), scale_of(p), zero_of(p));
            }
            store8(K + to, y);
        }
        if (V) {
            float y[8] = {};
            if (id >= 0) {
                uint32_t w[8];
                __builtin_memcpy(w, __builtin_assume_aligned(words, 16), 32);
                const uint32_t p = *reinterpret_cast<const uint32_t*>(block + kv.value_params() + (slot + i) * 4);
                const int shift = 4 * ((slot + i) & 7);
#pragma unroll
                for (int e = 0; e < 8; e++) y[e] = __builtin_fmaf((float)(w[e] >> shift & 15u), scale_of(p), zero_of(p));
            }
            store8(V + to, y);
        }
    }
}
// ---------------------------------------------------------------------------------------------------------- attention
//
// Scores and outputs come from v_mfma_f32_16x16x32_f16 on the codes themselves.  A float16 whose bits are a code c is the subnormal number
// c 2^-24, and c << 4 is c 2^-20: two codes become an operand word with one AND, four with one shift more.  The factor of 16 at every
// other element goes into the other operand.  A scale and a zero per token make
//     q . k_t = ks_t sum_d q_d c_td + kz_t sum_d q_d
//     sum_t p_t v_td = sum_t w_t c_td - 8 sum_t w_t + sum_t p_t (vz_t + 8 vs_t),   w_t = p_t vs_t
// with w_t rounded to float16 (where the result is float16: the sum of two) in both of its sums, so that its rounding only meets code - 8,
// which is what is rounded where values are multiplied.  The three sums grow with the length while what they make together does not: every 16 steps the second and
// third are joined to the first, which so holds outputs, and no other sum goes over more than 512 tokens (131072 tokens whose values cancel, about code 8 / about code 1:
// off by 3e-5 / 5e-4 of the weights with each sum by itself, now 1e-7 / 2e-6, for 4 % of a prompt's time; -8 as one more operand of each
// block of channels, so that no sum grows at all, costs 12 to 19 %).  Queries are scaled by a power of two so that their largest
// magnitude is in [2^14, 2^15): a float16 or bfloat16 keeps all of its bits, down to 2^-34 of the largest (2^-38 where codes do not count 16 times).  Weights have a unit of their own in
// each row, a power of two that follows the largest p vs that the row has met (not the largest vs: a token that the row does not see, or hardly, does not move it): that
// one is 2^6 or more, at most 2^15, and what is below 2^-27 of it is lost.  What weights are relative to is a power of two as well, so
// that both move without a rounding.
//
// A step is 32 tokens of one wavefront.  Keys are the A operand: row r of block b (two blocks of 16) is token 8 (r / 4) + 4 b + r % 4, so that
// lane quarter g ends with the scores of tokens 8 g .. 8 g + 7 of its column (a query), in the order in which the second product takes
// its weights as B operand: no lanes are exchanged.  The values of 8 tokens of a channel are one word of the cache, its A operand.
//
// What bounds it: of one token per sequence the cache's bytes (65003 tokens of 8 x 4 heads of 128: 21.3 us, 3.3 TB/s with two launches; 64 sequences of 2000 to
// 4000 43.5 us, 4.8 TB/s), with 8 heads of 64 per head of keys the vector ALU; of prompts the vector ALU, at 24 instructions per score of a wavefront beside two matrix
// instructions (2 x 2500 new of 4099, 8 x 4 heads of 128: 356 us, 0.5 PFLOP/s).
// Rows of a tile are (token, query head of the group) pairs of one sequence and one head of keys.

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));

// eight codes as operand words: word p holds elements p and p + 4, at 2^-24 for even p and 2^-20 for odd p
__device__ __forceinline__ v8h codes8(uint32_t w) {
    const uint32_t u = w >> 8;
    const v4u r = {w & 0x000F000Fu, w & 0x00F000F0u, u & 0x000F000Fu, u & 0x00F000F0u};
    return __builtin_bit_cast(v8h, r);
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    const v2f f = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, v2h));
}
__device__ __forceinline__ v2f unpack_f16(uint32_t w) { return __builtin_convertvector(__builtin_bit_cast(v2h, w), v2f); }

// the other lane quarters' values meet: fn(lanes' own and the 16 and then the 32 lanes across), the same in all quarters, without LDS
template <typename F>
__device__ __forceinline__ float over_quarters(float x, F&& fn) {
    const uint32_t a = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane16_swap(a, a, false, false);
    const uint32_t b = __builtin_bit_cast(uint32_t, fn(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1])));
    const auto q = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return fn(__builtin_bit_cast(float, (uint32_t)q[0]), __builtin_bit_cast(float, (uint32_t)q[1]));
}
__device__ __forceinline__ float max_over_quarters(float x) {
    return over_quarters(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float sum_over_quarters(float x) {
    return over_quarters(x, [](float a, float b) { return a + b; });
}

// a power of two from its biased exponent
__device__ __forceinline__ float power(int e) { return __builtin_bit_cast(float, (uint32_t)e << 23); }

constexpr int kMostSplits = 64;

struct Kv4Attend {
    Kv4 kv;
    Kv4Rows q;
    int heads_q, group, splits;
    float scale2;      // scale * log2(e)
    void* out;
    float* part;       // [splits][tokens * heads_q][dim], then [splits][tokens * heads_q][2]: sums, maximum (in powers of two) and sum of weights
};

// which tile of which sequence a workgroup's number is, with that sequence's rows of the call and its length; false behind the last
struct Kv4Tile {
    int s, tile, first, end, length, after;   // after: starts[s + 1]
};
__device__ __forceinline__ bool find_tile(const Kv4& kv, int group, int tile_rows, int number, Kv4Tile* t) {
    int before = 0;
    for (int b0 = 0; b0 < kv.sequences; b0 += 64) {
        const int b = min(b0 + lane_id(), kv.sequences - 1);
        const int from = kv.starts[b], to = kv.starts[b + 1], length = kv.lens[b], first = max(from, 0), end = min(to, kv.tokens);   // together: one wait
        const int64_t rows = b0 + lane_id() < kv.sequences ? (int64_t)max(0, end - first) * group : 0;
        const int tiles = (int)((uint32_t)(rows + tile_rows - 1) / (uint32_t)tile_rows);   // (below 2^31 rows in a call)
        int sum = tiles;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int o = __shfl_up(sum, d);
            if (lane_id() >= d) sum += o;
        }
        const uint64_t past = __ballot(before + sum > number);
        if (past) {
            const int l = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)past) - 1);
            auto at = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
            *t = {b0 + l, at(sum) - 1 - (number - before), at(first), at(end), at(length), at(to)};   // the last tiles, which see most, first
            return true;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}

// One sequence and head of the cache as the steps read it.  A lane each holds 64 entries of the table at a time, so that no step waits for an entry before
// it can ask for its codes (two prompts of 2500 tokens, 4 x 8 heads of 128, 680 -> 597 us).  Positions and offsets in a page are 32 bits, pages are
// found in 64.
struct Kv4Pages {
    const int32_t* table;
    const char* cache;     // of the head
    uint32_t page_bytes;
    int pages, width, shift, mask;   // mask: page - 1
    int window = 0, ids;             // ids: entry window + lane, -1 outside of the cache

    __device__ __forceinline__ void look(int i) {
        window = i;
        const int at = window + lane_id(), id = table[min(at, width - 1)];
        ids = at < width && (uint32_t)id < (uint32_t)pages ? id : -1;
    }
    __device__ __forceinline__ int id(int i) {   // i the same in all lanes, not falling
        if (i - window >= 64) look(i);
        return __builtin_amdgcn_readlane(ids, i - window);
    }
    __device__ __forceinline__ const char* page(int id) const { return cache + (uint64_t)(uint32_t)max(id, 0) * page_bytes; }
    // whether entries first .. last are all pages of the cache
    __device__ __forceinline__ bool all_there(int first, int last) const {
        bool good = last < width && (window > first || window + lane_id() > last || ids >= 0);
        for (int i = window > first ? first : window + 64; i <= last; i += 64) {
            const int id = table[min(min(i + lane_id(), last), width - 1)];
            good &= (uint32_t)id < (uint32_t)pages;
        }
        return __all(good);
    }
};
// where a step's tokens lie: two pages where those hold 16
struct Kv4Place {
    const char *first, *second;
    bool first_there, second_there;
    __device__ __forceinline__ const char* of(int eight) const { return eight >> 1 ? second : first; }   // the page of tokens 8 eight ..
};
__device__ __forceinline__ Kv4Place place_of(Kv4Pages& q, int t0) {
    const int i = t0 >> q.shift, a = q.id(i), b = q.shift >= 5 ? a : q.id(i + 1);
    return {q.page(a), q.page(b), a >= 0, b >= 0};
}

// what a step of 32 tokens takes from the cache
template <int D>
struct Kv4Step {
    uint32_t kw[2][D / 32], vw[D / 16], kp[8], vp[8];
    bool there;   // the page of the lane's tokens 8 g .. 8 g + 7

    __device__ __forceinline__ void fetch_keys(const Kv4Pages& q, const Kv4Place& p, int t0, int c, int g) {
        // codes: this lane's row of each block; (scale, zero): tokens 8 g .. 8 g + 7
        const int kt = t0 + 8 * (c >> 2) + (c & 3), pt = t0 + 8 * g;   // + 4 for the second block
        const char* const kb = p.of(c >> 2) + (uint32_t)((kt & q.mask) * (D / 2) + g * (D / 8));
        const char* const pb = p.of(g) + (uint32_t)((q.mask + 1) * D + (pt & q.mask) * 4);
        __builtin_memcpy(kw[0], __builtin_assume_aligned(kb, 4), D / 8);
        __builtin_memcpy(kw[1], __builtin_assume_aligned(kb + 4 * (D / 2), 4), D / 8);
        __builtin_memcpy(kp, __builtin_assume_aligned(pb, 16), 32);
    }
    __device__ __forceinline__ void fetch_values(const Kv4Pages& q, const Kv4Place& p, int t0, int c, int g) {
        const int slot = (t0 + 8 * g) & q.mask;
        there = g >> 1 ? p.second_there : p.first_there;
        const char* const b = p.of(g);
        __builtin_memcpy(vw, __builtin_assume_aligned(b + (uint32_t)((q.mask + 1) * (D / 2) + (slot / 8 * D + c * (D / 16)) * 4), 8), D / 4);
        __builtin_memcpy(vp, __builtin_assume_aligned(b + (uint32_t)((q.mask + 1) * (D + 4) + slot * 4), 16), 32);
    }
};

// CB blocks of 16 rows per wavefront.  WT = 4: the wavefronts of a workgroup split the tokens of one tile and meet in LDS; WT = 1: they have tiles of
// their own side by side.
template <typename T, int D, int CB, int WT>
__global__ __launch_bounds__(WT == 1 ? 256 : 64 * WT, D * CB <= 256 && D < 256 ? 2 : 1) void k_kv4_attend(Kv4Attend p) {
    constexpr int PARTS = std::is_same<T, _Float16>::value ? 2 : 1, ND = D / 32, NB = D / 16, TILE = 16 * CB, WG_ROWS = WT == 1 ? TILE * 4 : TILE;
    extern __shared__ __align__(16) float lds[];   // WT = 4: [4][16 CB][D + 4] sums, then [4][16 CB][2]; WT = 1: the wavefronts' queries as operands, [4][CB][ND][64] of 16 bytes
    const Kv4& kv = p.kv;
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    Kv4Tile found;
    if (!find_tile(kv, p.group, WG_ROWS, blockIdx.x, &found)) return;   // (the whole workgroup)
    const int s = found.s, tile = found.tile;
    const int head = blockIdx.y, split = blockIdx.z;
    const int first = found.first, n = found.end - first;
    const int held = min(max(found.length, 0), kv.width << kv.shift);   // (at most 2^30 tokens, by the host's check)
    const uint32_t rows = (uint32_t)n * p.group, group = p.group;   // (a call has fewer than 2^31 query rows)
    const int64_t base = (int64_t)found.length - found.after + first;   // position of the call's first token
    const uint32_t row0 = (uint32_t)tile * WG_ROWS + (WT == 1 ? wave * TILE : 0);
    if (WT == 1 && row0 >= rows) return;
    const uint32_t last_row = min(row0 + TILE, rows) - 1;
    const int most = (int)max((int64_t)0, min((int64_t)held, base + last_row / group + 1)), least = (int)max((int64_t)0, min((int64_t)held, base + row0 / group + 1));
    const int steps = (most + 31) / 32, per = (steps + p.splits - 1) / p.splits, from = per * split, to = min(steps, from + per);
    Kv4Pages seq = {kv.table + s * kv.table_stride, kv.cache + head * kv.head_bytes, (uint32_t)kv.page_bytes, (int)kv.pages, kv.width, kv.shift, kv.page - 1};
    seq.look((from * 32) >> kv.shift);
    // the first codes are asked for ahead of the queries.  Of few rows memory is what counts: the codes of the next steps are on their way while one is
    // computed; of many, the next step's keys when this one's scores are there, its values when this one's sums are
    constexpr int AHEAD = WT == 1 ? 1 : D <= 128 ? 3 : 2;
    Kv4Step<D> ring[AHEAD];
    int st = from + (WT == 1 ? 0 : wave);
    auto fetch = [&](Kv4Step<D>& x, int step) {
        const Kv4Place at = place_of(seq, step * 32);
        x.fetch_keys(seq, at, step * 32, c, g), x.fetch_values(seq, at, step * 32, c, g);
    };
#pragma unroll
    for (int i = 0; i < AHEAD; i++)
        if (st + i * WT < to) fetch(ring[i], st + i * WT);
    // rows: (token, query head of the group); what a row sees: tokens before `seen`
    int seen[CB];
    constexpr bool KEPT = WT > 1;   // queries stay in registers; of many rows they lie in LDS: with them two wavefronts per SIMD do not fit (597 -> 500 us)
    v8h q[KEPT ? CB : 1][KEPT ? ND : 1];
    v4u* const mine_q = reinterpret_cast<v4u*>(lds) + (size_t)wave * CB * ND * 64 + lane;
    float qsum[CB], unit[CB];   // sum of the scaled queries in units of the products; powers of two per unit of score
#pragma unroll
    for (int b = 0; b < CB; b++) {
        const uint32_t row = min(row0 + 16 * b + c, rows - 1);
        const int j = (int)(row / group), hq = head * p.group + (int)(row % group);
        seen[b] = (int)max((int64_t)0, min((int64_t)held, base + j + 1));
        const T* const from = static_cast<const T*>(p.q.p) + (int64_t)(first + j) * p.q.token_stride + (int64_t)hq * p.q.head_stride + g * (D / 4);
        float x[ND][8], top = 0.0f, sum = 0.0f;
#pragma unroll
        for (int i = 0; i < ND; i++) {
            load8(from + 8 * i, x[i]);
#pragma unroll
            for (int e = 0; e < 8; e++) top = fmaxf(top, __builtin_fabsf(x[i][e])), sum += x[i][e];
        }
        top = max_over_quarters(top), sum = sum_over_quarters(sum);
        const int up = 141 - min(max((int)(__builtin_bit_cast(uint32_t, top) >> 23), 27), 254);   // times 2^up the largest is in [2^14, 2^15)
#pragma unroll
        for (int i = 0; i < ND; i++) {
            v4u h;
#pragma unroll
            for (int w = 0; w < 4; w++) {
                h[w] = pack_f16(__builtin_ldexpf(x[i][w], up - 4 * (w & 1)), __builtin_ldexpf(x[i][w + 4], up - 4 * (w & 1)));
            }
            if constexpr (KEPT) q[b][i] = __builtin_bit_cast(v8h, h);
            else mine_q[(b * ND + i) * 64] = h;
        }
        qsum[b] = __builtin_ldexpf(sum, up - 24);   // scores are in units of 2^(24 - up)
        unit[b] = fminf(fmaxf(__builtin_ldexpf(p.scale2, 24 - up), 0x1p-126f), 0x1.fffffep127f);
    }
    v4f o[CB][NB], wsum[CB];
    float m[CB], limit[CB], l[CB], zsum[CB];   // m: what the weights are relative to, a whole power of two
    float one[CB];                             // what a weight of 1 (times kScales) is in float16, a power of two: the rows' units
#pragma unroll
    for (int b = 0; b < CB; b++) {
#pragma unroll
        for (int i = 0; i < NB; i++) o[b][i] = v4f{0, 0, 0, 0};
        wsum[b] = v4f{0, 0, 0, 0}, m[b] = limit[b] = -__builtin_inff(), l[b] = zsum[b] = 0.0f, one[b] = power(254);
    }
    const v4u eights = {0x00080008u, 0x00800080u, 0x00080008u, 0x00800080u};   // 8 in units of the codes
    constexpr float kScales = 0x1p-12f;   // times the largest scale a weight of 2^8 is a float
    auto exponent = [](float x) { return (int)(__builtin_bit_cast(uint32_t, x) >> 23); };   // biased, of x >= 0

    // EDGE: some row does not see all of the step's tokens
    // keys_done, values_done: called when those of the step are not needed any more
    auto compute = [&](Kv4Step<D>& x, int t0, auto edge, auto keys_done, auto values_done) {
        constexpr bool EDGE = decltype(edge)::value;
        float vs[8], vz[8];
        if (EDGE) {
#pragma unroll
            for (int e = 0; e < 8; e++) x.vp[e] = x.there && t0 + 8 * g + e < held ? x.vp[e] : 0u;   // behind the sequence: not looked at
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float sc = scale_of(x.vp[e]);
            vz[e] = __builtin_fmaf(8.0f, sc, zero_of(x.vp[e]));
            vs[e] = sc * ((e & 1) ? kScales / 16 : kScales);
        }
        float sc[CB][8];
        {
            v4f a[2][CB];
#pragma unroll
            for (int i = 0; i < ND; i++) {
                const v8h k0 = codes8(x.kw[0][i]), k1 = codes8(x.kw[1][i]);
#pragma unroll
                for (int cb = 0; cb < CB; cb++) {
                    v8h qi;
                    if constexpr (KEPT) qi = q[cb][i];
                    else qi = __builtin_bit_cast(v8h, mine_q[(cb * ND + i) * 64]);
                    if (i == 0) a[0][cb] = a[1][cb] = v4f{0, 0, 0, 0};
                    a[0][cb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qi, a[0][cb], 0, 0, 0);
                    a[1][cb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qi, a[1][cb], 0, 0, 0);
                }
            }
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float ks = scale_of(x.kp[4 * b + e]), kz = zero_of(x.kp[4 * b + e]);
#pragma unroll
                    for (int cb = 0; cb < CB; cb++) sc[cb][4 * b + e] = __builtin_fmaf(a[b][cb][e], ks, qsum[cb] * kz);
                }
        }
        __builtin_amdgcn_sched_barrier(0);
        keys_done();
        if ((t0 / (32 * WT)) % 16 == 0) {
#pragma unroll
            for (int cb = 0; cb < CB; cb++) {
                const float z = sum_over_quarters(zsum[cb]);
                int held = exponent(one[cb]);
                if (__any(exponent(__builtin_fabsf(z)) + held > 390)) {   // z in the row's unit is 2^100 or more: the unit goes down, weights hardly count beside it
                    const int high = exponent(__builtin_fabsf(z)), next = high + held > 390 ? 350 - high : held;
                    const float fo = __builtin_ldexpf(1.0f, next - held);
                    wsum[cb] *= fo;
#pragma unroll
                    for (int i = 0; i < NB; i++) o[cb][i] *= fo;
                    one[cb] = power(next), held = next;
                }
                const v4f d = __builtin_ldexpf(z, held - 163) - wsum[cb];
#pragma unroll
                for (int i = 0; i < NB; i++) o[cb][i] += d;
                wsum[cb] = v4f{0, 0, 0, 0}, zsum[cb] = 0.0f;
            }
        }
        v8h wh[CB], wl[PARTS == 2 ? CB : 1];
#pragma unroll
        for (int cb = 0; cb < CB; cb++) {
            if (EDGE) {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (!x.there || t0 + 8 * g + e >= seen[cb]) sc[cb][e] = -__builtin_inff();
            }
            float top = sc[cb][0];
#pragma unroll
            for (int e = 1; e < 8; e++) top = fmaxf(top, sc[cb][e]);
            // what the weights are relative to moves when it is passed by more than 2^8 (and by the first tokens that a row sees): they and their sums
            // have room for that, and most steps need not touch the sums (500 -> 364 us, with the steps that look at each token in a loop of their own)
            if (__any(top * unit[cb] > limit[cb])) {
                const float reach = max_over_quarters(top) * unit[cb];
                const bool move = reach > limit[cb];
                const float to = move ? __builtin_ceilf(reach) : m[cb];
                const int by = move ? (int)fminf(to - m[cb], 512.0f) : 0;   // the row's unit goes up with it, as far as it may
                const int held = exponent(one[cb]), next = min(held + by, 254);
                const float f = __builtin_ldexpf(1.0f, -by), fo = __builtin_ldexpf(1.0f, next - held - by);
                l[cb] *= f, zsum[cb] *= f, wsum[cb] *= fo;
#pragma unroll
                for (int i = 0; i < NB; i++) o[cb][i] *= fo;
                m[cb] = to, limit[cb] = to + 8.0f, one[cb] = power(next);
            }
            const float off = m[cb] == -__builtin_inff() ? 0.0f : -m[cb];
            uint32_t hi[4], lo[4];
            float w[8], most = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[cb][e], unit[cb], off));
                l[cb] += y;
                const bool hidden = EDGE && (!x.there || t0 + 8 * g + e >= seen[cb]);   // what a row does not see may be no number
                zsum[cb] = hidden ? zsum[cb] : __builtin_fmaf(y, vz[e], zsum[cb]);
                w[e] = hidden ? 0.0f : y * vs[e];
                most = fmaxf(most, __builtin_fabsf(w[e]));   // (NaN, of a token of NaN, is passed over)
            }
            if (__any(most * one[cb] > 0x1p15f)) {   // the row's unit goes down
                most = max_over_quarters(most);
                const int held = exponent(one[cb]), next = most * one[cb] > 0x1p15f ? 260 - min(exponent(most), 254) : held;
                const float fo = __builtin_ldexpf(1.0f, next - held);
                wsum[cb] *= fo;
#pragma unroll
                for (int i = 0; i < NB; i++) o[cb][i] *= fo;
                one[cb] = power(next);
            }
#pragma unroll
            for (int e = 0; e < 8; e++) w[e] *= one[cb];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                hi[e] = pack_f16(w[e], w[e + 4]);
                if (PARTS == 2) {
                    const v2f h = unpack_f16(hi[e]);
                    lo[e] = pack_f16(w[e] - h[0], w[e + 4] - h[1]);
                }
            }
            wh[cb] = __builtin_bit_cast(v8h, (v4u{hi[0], hi[1], hi[2], hi[3]}));
            if (PARTS == 2) wl[PARTS == 2 ? cb : 0] = __builtin_bit_cast(v8h, (v4u{lo[0], lo[1], lo[2], lo[3]}));
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i <= NB; i++) {
            const v8h a = i == NB ? __builtin_bit_cast(v8h, eights) : codes8(x.vw[i == NB ? 0 : i]);
#pragma unroll
            for (int cb = 0; cb < CB; cb++) {
                v4f& to = i == NB ? wsum[cb] : o[cb][i == NB ? 0 : i];
                to = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, wh[cb], to, 0, 0, 0);
                if (PARTS == 2) to = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, wl[PARTS == 2 ? cb : 0], to, 0, 0, 0);
            }
        }
        values_done();
    };
    // Steps below `plain` are seen by all rows, in pages of the cache.  What is left, the last step or two, looks at each token; so does everything where
    // the table has a bad page before (what it holds behind them does not count: 48 sequences of 5002 tokens in pages of 16, -1 behind, 63 -> 56 us).
    const int whole = min(to, least / 32), plain = from < whole && seq.all_there((from * 32) >> kv.shift, (whole * 32 - 1) >> kv.shift) ? whole : 0;
    auto nothing = []() {};
    if constexpr (WT == 1) {
        Kv4Place at;
        auto keys = [&]() {
            if (st + 1 < to) at = place_of(seq, (st + 1) * 32), ring[0].fetch_keys(seq, at, (st + 1) * 32, c, g);
        };
        auto values = [&]() {
            if (st + 1 < to) ring[0].fetch_values(seq, at, (st + 1) * 32, c, g);
        };
        for (; st < plain; st++) compute(ring[0], st * 32, std::false_type{}, keys, values);
        for (; st < to; st++) compute(ring[0], st * 32, std::true_type{}, keys, values);
    } else {
        for (; st + (AHEAD - 1) * WT < plain; st += AHEAD * WT)
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                compute(ring[i], (st + i * WT) * 32, std::false_type{}, nothing, nothing);
                if (st + (i + AHEAD) * WT < to) fetch(ring[i], st + (i + AHEAD) * WT);
            }
        for (; st < to; st += AHEAD * WT)
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                if (st + i * WT < to) compute(ring[i], (st + i * WT) * 32, std::true_type{}, nothing, nothing);
                if (st + (i + AHEAD) * WT < to) fetch(ring[i], st + (i + AHEAD) * WT);
            }
    }
    // channel (4 g + e) NB + i of a row is in accumulator e of block i
    auto row_at = [&](uint32_t r) { return (int64_t)(first + (int)(r / group)) * p.heads_q + head * p.group + (int)(r % group); };
#pragma unroll
    for (int b = 0; b < CB; b++) {
        const int back = 163 - exponent(one[b]);   // of the row's unit, kScales and the codes: 2^(127 + 12 + 24 - exponent)
        l[b] = sum_over_quarters(l[b]), zsum[b] = sum_over_quarters(zsum[b]);
        if constexpr (WT == 1) {
            const uint32_t r = row0 + 16 * b + c;
            if (r >= rows) continue;
            const int64_t at = row_at(r);
            const float f = l[b] == 0.0f ? 0.0f : 1.0f / l[b];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                T v[NB];
#pragma unroll
                for (int i = 0; i < NB; i++) v[i] = (T)(l[b] == 0.0f ? 0.0f : (__builtin_ldexpf(o[b][i][e] - wsum[b][e], back) + zsum[b]) * f);
                __builtin_memcpy(static_cast<T*>(p.out) + at * D + (4 * g + e) * NB, v, sizeof(v));
            }
        } else {   // the wavefronts meet
            constexpr int LD = D + 4;
            float* const mine = lds + (wave * TILE + 16 * b + c) * LD;
#pragma unroll
            for (int i = 0; i < NB; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) mine[(4 * g + e) * NB + i] = __builtin_ldexpf(o[b][i][e] - wsum[b][e], back) + zsum[b];
            float* const ml = lds + WT * TILE * LD;
            if (g == 0) ml[(wave * TILE + 16 * b + c) * 2] = m[b], ml[(wave * TILE + 16 * b + c) * 2 + 1] = l[b];
        }
    }
    if constexpr (WT > 1) {
        constexpr int LD = D + 4;
        const int64_t all = (int64_t)kv.tokens * p.heads_q;
        const float* const ml = lds + WT * TILE * LD;
        __syncthreads();
        // 16 lanes to a row, NB channels each
        const int r = threadIdx.x >> 4, d = (threadIdx.x & 15) * NB;
        static_assert(WT * 64 == 16 * TILE, "a lane per NB channels of the tile");
        const uint32_t rr = row0 + r;
        if (rr >= rows) return;
        float top = -__builtin_inff(), den = 0.0f, f[WT], sum[NB] = {};
#pragma unroll
        for (int w = 0; w < WT; w++) top = fmaxf(top, ml[(w * TILE + r) * 2]);
#pragma unroll
        for (int w = 0; w < WT; w++) {
            const float lw = ml[(w * TILE + r) * 2 + 1];
            f[w] = lw == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(ml[(w * TILE + r) * 2] - top);   // (sums without weights are zeros)
            den = __builtin_fmaf(lw, f[w], den);
        }
#pragma unroll
        for (int w = 0; w < WT; w++)
#pragma unroll
            for (int i = 0; i < NB; i++) sum[i] = __builtin_fmaf(lds[(w * TILE + r) * LD + d + i], f[w], sum[i]);
        const int64_t at = row_at(rr);
        if (p.splits == 1) {
            T y[NB];
#pragma unroll
            for (int i = 0; i < NB; i++) y[i] = (T)(den == 0.0f ? 0.0f : sum[i] / den);
            __builtin_memcpy(static_cast<T*>(p.out) + at * D + d, y, sizeof(y));
        } else {
            __builtin_memcpy(p.part + (split * all + at) * D + d, sum, sizeof(sum));
            if (d == 0) {
                float* const pm = p.part + p.splits * all * D + (split * all + at) * 2;
                pm[0] = top, pm[1] = den;
            }
        }
    }
}

// The parts of a row meet: a workgroup per row, D / 4 lanes on its channels, so that 256 / (D / 4) parts are read at a time.  A launch and three dependent
// loads: 3 us.
template <typename T, int D>
__global__ __launch_bounds__(256) void k_kv4_join(Kv4Attend p) {
    constexpr int LANES = D / 4, GROUPS = 256 / LANES;
    __shared__ v4f sums[GROUPS][LANES];
    __shared__ float weight[64], total;
    const int64_t all = (int64_t)p.kv.tokens * p.heads_q, at = blockIdx.x;
    const int token = (int)((uint32_t)at / (uint32_t)p.heads_q);   // (below 2^31 rows)
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    static_assert(kMostSplits <= 64, "a lane per part");
    // what all depends on is asked for at once: the first parts before their weights are known
    const float* const pm = p.part + p.splits * all * D;
    const bool mine = (int)threadIdx.x < p.splits;   // (the first wavefront's lanes)
    const float m = mine ? pm[(threadIdx.x * all + at) * 2] : -__builtin_inff(), l = mine ? pm[(threadIdx.x * all + at) * 2 + 1] : 0.0f;
    constexpr int EARLY = 4;
    v4f x[EARLY];
#pragma unroll
    for (int i = 0; i < EARLY; i++) x[i] = *reinterpret_cast<const v4f*>(p.part + (min(group + i * GROUPS, p.splits - 1) * all + at) * D + 4 * lane);
    if (token < p.kv.starts[0] || token >= p.kv.starts[p.kv.sequences]) return;   // (the whole workgroup)
    if (threadIdx.x < 64) {
        float top = m;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
        const float w = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m - top);
        float den = w * l;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) den += __shfl_xor(den, d);
        weight[threadIdx.x] = w;
        if (threadIdx.x == 0) total = den;
    }
    __syncthreads();
    v4f sum = {0, 0, 0, 0};
    if (group < GROUPS) {
#pragma unroll
        for (int i = 0; i < EARLY; i++) {
            const float w = group + i * GROUPS < p.splits ? weight[group + i * GROUPS] : 0.0f;
            sum += w == 0.0f ? v4f{0, 0, 0, 0} : w * x[i];
        }
        for (int i = group + EARLY * GROUPS; i < p.splits; i += GROUPS) {
            const v4f y = *reinterpret_cast<const v4f*>(p.part + (i * all + at) * D + 4 * lane);
            const float w = weight[i];
            sum += w == 0.0f ? v4f{0, 0, 0, 0} : w * y;
        }
        sums[group][lane] = sum;
    }
    __syncthreads();
    if (threadIdx.x >= LANES) return;
#pragma unroll
    for (int i = 1; i < GROUPS; i++) sum += sums[i][lane];
    T y[4];
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = (T)(total == 0.0f ? 0.0f : sum[e] / total);
    __builtin_memcpy(static_cast<T*>(p.out) + at * D + 4 * lane, y, sizeof(y));
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

// How a call is split: tiles of 16 rows, whose tokens the four wavefronts of a workgroup share, or wavefronts of 32 rows (16 of dim 256) on all tokens, which
// read and unpack the cache once for twice the rows and have no sums to join.  Fewer workgroups of the first kind than run at once (two per compute
// unit, one of dim 256) split their tokens further, down to 512 each, and a second launch joins the parts.  The choice goes by an estimate in us: a workgroup
// costs 6 and a step of 32 tokens of a wavefront `narrow` or `wide`; fitted to 8 heads of 4 x 128 at 4000 tokens, 16 / 32 rows measured: 512 new 83 / 167,
// 1024 156 / 186, 2048 247 / 217, 4 x 512 at 2000 126 / 109, 512 at 512 23.5 / 25.9; of dim 256, 4 heads: 1000 new 174 / 184.
struct Kv4Plan {
    int blocks, waves;   // CB, WT
    int64_t tiles;
    int splits;
};
int64_t tiles_of(const ftnn_kv4_t& kv, int group, int rows) {   // at most: tokens of a sequence share tiles, sequences do not
    const int64_t t = kv.tokens;
    return std::min((t * group + rows - 1) / rows + kv.sequences, t * ((group + rows - 1) / rows));
}
Kv4Plan plan_of(const ftnn_kv4_t& kv, int heads_q, int max_len) {
    const int group = heads_q / kv.heads, blocks = kv.dim <= 128 ? 2 : 1;
    const int64_t capacity = (int64_t)kv.width * kv.page, most = max_len > 0 ? std::min<int64_t>(max_len, capacity) : capacity;
    const int64_t resident = kv.dim == 256 ? 240 : 512;
    const int64_t wide = tiles_of(kv, group, 64 * blocks), narrow = tiles_of(kv, group, 16), spread = std::max<int64_t>(1, narrow * kv.heads);
    const int splits = (int)std::max<int64_t>(1, std::min<int64_t>({resident / spread, (most + 511) / 512, kMostSplits}));
    const double narrow_step = kv.dim == 64 ? 0.8 : kv.dim <= 128 ? 1.1 : 1.2, wide_step = kv.dim == 64 ? 1.2 : kv.dim <= 128 ? 1.6 : 1.45;
    const double steps = std::max(1.0, ((double)most - 0.5 * kv.tokens / std::max(kv.sequences, 1)) / 32);   // of a row, in the mean
    auto rounds = [&](int64_t workgroups, int64_t at_once) { return (double)((workgroups + at_once - 1) / at_once); };
    const double by16 = rounds(spread * splits, resident) * (6 + std::max(1.0, steps / 4 / splits) * narrow_step) + (splits > 1 ? 5 : 0);
    const double by32 = rounds(wide * kv.heads, 512) * (6 + steps * wide_step);
    if (by32 < by16) return {blocks, 1, wide, 1};
    return {1, 4, narrow, splits};
}

constexpr int kMostWorkgroups = 1 << 24;   // of 256 threads along a side: a launch holds fewer than 2^32

}  // namespace

hipError_t launch_kv4_append(const ftnn_kv4_t& kv, int dtype, const Kv4Rows& k, const Kv4Rows& v, const Kv4Rotation& r, int heads_q,
                             const Kv4Rows& q, void* d_q_out, hipStream_t st) {
    const Kv4 dv = device_view(kv);
    const int eights = eights_of(kv), groups = (kv.heads + heads_q + 3) / 4;
    if (eights >= kMostWorkgroups) return hipErrorInvalidConfiguration;
    const int heads_at_a_time = std::max(1, std::min(groups, (512 + eights - 1) / eights));   // about two workgroups per compute unit, or all there are
    return with_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        return with_dim(kv.dim, [&](auto d) {
            k_kv4_append<T, decltype(d)::value><<<dim3(eights, heads_at_a_time), dim3(256), 0, st>>>(dv, k, v, r, heads_q, q, static_cast<T*>(d_q_out));
            return hipGetLastError();
        });
    });
}

hipError_t launch_kv4_read(const ftnn_kv4_t& kv, int dtype, void* d_k, void* d_v, hipStream_t st) {
    const Kv4 dv = device_view(kv);
    if (eights_of(kv) >= kMostWorkgroups) return hipErrorInvalidConfiguration;
    return with_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        return with_dim(kv.dim, [&](auto d) {
            k_kv4_read<T, decltype(d)::value><<<dim3(eights_of(kv), (kv.heads + 3) / 4), dim3(256), 0, st>>>(dv, static_cast<T*>(d_k), static_cast<T*>(d_v));
            return hipGetLastError();
        });
    });
}

int64_t kv4_attention_scratch(const ftnn_kv4_t& kv, int heads_q, int max_len) {
    const int64_t splits = plan_of(kv, heads_q, max_len).splits;
    return splits == 1 ? 0 : splits * kv.tokens * heads_q * (kv.dim + 2) * 4;
}

hipError_t launch_kv4_attention(const ftnn_kv4_t& kv, int dtype, int heads_q, const Kv4Rows& q, float scale, int max_len, void* d_out,
                                void* d_scratch, hipStream_t st) {
    const Kv4Plan plan = plan_of(kv, heads_q, max_len);
    if (plan.tiles >= kMostWorkgroups) return hipErrorInvalidConfiguration;
    Kv4Attend p;
    p.kv = device_view(kv), p.q = q, p.heads_q = heads_q, p.group = heads_q / kv.heads, p.splits = plan.splits;
    p.scale2 = scale * 1.44269504088896341f, p.out = d_out, p.part = static_cast<float*>(d_scratch);
    auto go = [&](auto t) {
        typedef decltype(t) T;
        return with_dim(kv.dim, [&](auto d) {
            constexpr int D = decltype(d)::value;
            auto run = [&](auto cb, auto wt) {
                constexpr int CB = decltype(cb)::value, WT = decltype(wt)::value, bytes = WT == 1 ? 4 * CB * (D / 32) * 1024 : WT * 16 * CB * (D + 4 + 2) * 4;
                auto* const kern = k_kv4_attend<T, D, CB, WT>;
                static const hipError_t set = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, std::max(bytes, 16));
                if (set != hipSuccess) return set;
                kern<<<dim3((unsigned)plan.tiles, kv.heads, plan.splits), dim3(WT == 1 ? 256 : 64 * WT), bytes, st>>>(p);
                return hipGetLastError();
            };
            using One = std::integral_constant<int, 1>;
            using Two = std::integral_constant<int, 2>;
            hipError_t e;
            if (plan.waves == 4) e = run(One{}, std::integral_constant<int, 4>{});
            else if constexpr (D <= 128) e = run(Two{}, One{});
            else e = run(One{}, One{});
            if (e != hipSuccess || p.splits == 1) return e;
            k_kv4_join<T, D><<<dim3((unsigned)((int64_t)kv.tokens * heads_q)), dim3(256), 0, st>>>(p);
            return hipGetLastError();
        });
    };
    return dtype == FTNN_F16 ? go((_Float16)0.0f) : go((__bf16)0.0f);
}

}  // namespace ftnn
