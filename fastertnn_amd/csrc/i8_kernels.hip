// Rows of 8-bit codes with a scale each, and their products with 8-bit and with packed ternary or binary weights.
#include <algorithm>

#include "tokens_internal.h"

namespace ftnn {

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef unsigned int v4u __attribute__((ext_vector_type(4)));
typedef unsigned short v8us __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------------------------------------ rows to 8-bit codes
//
// q = x * 127 / max|x|, rounded to the nearest integer, ties to even.  Codes next to a border have to come out as the formula says
// and not as 24 bits happen to: with x and max|x| of 24 bits each, a quotient that is no tie is at least 2^-32 of itself away from
// one (254 X and (2 k + 1) A are whole numbers in the same unit), 2^-33 at the first border, 1/2.  In 64 bits the product with
// the reciprocal is off by less than 2^-45; rounded to multiples of 2^-40 (what adding 1.5 * 2^12 does) ties become exact and
// others stay on their side.  Adding 1.5 * 2^52 then rounds to an integer, whose lowest byte is the code.  On this chip a 64-bit
// multiply-add issues at the rate of a 32-bit one, so this costs three instructions per value beside the loads.
//
// A row is read once: its values stay in registers between the maximum and the codes, up to NV vectors of 16 bytes per thread; what
// is beyond that is read again.

template <typename T>
struct Vec {   // 16 bytes of T
    static constexpr int N = 16 / sizeof(T);
    v4u w;
    __device__ __forceinline__ double at(int i) const {
        if constexpr (std::is_same<T, float>::value) {
            const uint32_t bits = w[i];   // (a bit cast of the element itself reads element 0)
            return (double)__builtin_bit_cast(float, bits);
        } else if constexpr (std::is_same<T, __bf16>::value) {
            return (double)__builtin_bit_cast(float, (i & 1) ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
        } else {
            return (double)(float)__builtin_bit_cast(_Float16, (unsigned short)(w[i / 2] >> (16 * (i & 1))));
        }
    }
    // the largest magnitude so far as a bit pattern: those of one sign order like whole numbers, infinity and NaN on top
    __device__ __forceinline__ void most(v4u& m) const {
        if constexpr (std::is_same<T, float>::value) {
            m = __builtin_elementwise_max(m, w & 0x7FFFFFFFu);
        } else {
            m = __builtin_bit_cast(v4u, __builtin_elementwise_max(__builtin_bit_cast(v8us, m), __builtin_bit_cast(v8us, w & 0x7FFF7FFFu)));
        }
    }
};
template <typename T>
__device__ __forceinline__ uint32_t most_of(const v4u& m) {
    if constexpr (std::is_same<T, float>::value) return max(max(m[0], m[1]), max(m[2], m[3]));
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) r = max(r, max(m[i] & 0xFFFFu, m[i] >> 16));
    return r;
}
template <typename T>
__device__ __forceinline__ float magnitude(uint32_t bits) {
    if constexpr (std::is_same<T, float>::value) return __builtin_bit_cast(float, bits);
    else if constexpr (std::is_same<T, __bf16>::value) return __builtin_bit_cast(float, bits << 16);
    else return (float)__builtin_bit_cast(_Float16, (unsigned short)bits);
}

// vector `c` of a row of K values; past the K-th zeros
template <typename T>
__device__ __forceinline__ Vec<T> load_vec(const T* row, int c, int K) {
    constexpr int N = Vec<T>::N;
    Vec<T> v;
    if ((c + 1) * N <= K) {
        __builtin_memcpy(&v.w, row + (size_t)c * N, 16);   // rows may start at any value: unaligned wide loads
    } else {
        T e[N];
#pragma unroll
        for (int i = 0; i < N; i++) e[i] = c * N + i < K ? row[(size_t)c * N + i] : (T)0.0f;
        __builtin_memcpy(&v.w, e, 16);
    }
    return v;
}

// ROWS rows per workgroup, W wavefronts on each
template <typename T, int W, int ROWS, int NV>
__global__ __launch_bounds__(64 * W * ROWS) void k_quantize_rows(const T* __restrict__ X, int64_t x_stride, int64_t rows, int K,
                                                                 int8_t* __restrict__ Q, int64_t q_stride, float* __restrict__ S) {
    constexpr int N = Vec<T>::N, TR = 64 * W;
    __shared__ uint32_t part[W * ROWS];
    const int sub = threadIdx.x / TR, t = threadIdx.x % TR;
    const int64_t row = (int64_t)blockIdx.x * ROWS + sub;
    const bool live = row < rows;   // all of a wavefront
    const T* const x = X + (live ? row : 0) * x_stride;
    const int nvec = ((K + 15) / 16) * 16 / N;   // with the zeros up to a whole 16
    Vec<T> v[NV];
    v4u m = {0, 0, 0, 0};
    if (live) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = i * TR + t;
            if (c < nvec) {
                v[i] = load_vec(x, c, K);
            } else {
                v[i].w = v4u{0, 0, 0, 0};
            }
        }
#pragma unroll
        for (int i = 0; i < NV; i++) v[i].most(m);
        for (int c = NV * TR + t; c < nvec; c += TR) load_vec(x, c, K).most(m);
    }
    uint32_t most = most_of<T>(m);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) most = max(most, (uint32_t)__shfl_xor((int)most, d));
    if constexpr (W > 1) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x / 64] = most;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < W; i++) most = max(most, part[sub * W + i]);
    }
    if (!live) return;
    const float top = magnitude<T>(most);
    const bool fine = top < __builtin_inff();   // neither NaN nor infinite
    const double inv = fine && top > 0.0f ? 127.0 / (double)top : 0.0;
    const uint32_t keep = fine ? 0xFFFFFFFFu : 0u;
    if (t == 0) S[row] = fine ? top / 127.0f : __builtin_nanf("");
    int8_t* const q = Q + row * q_stride;
    auto put = [&](const Vec<T>& w, int c) {
        uint32_t d[N / 4];
#pragma unroll
        for (int j = 0; j < N / 4; j++) {
            uint32_t b[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const double r = __builtin_fma(w.at(4 * j + i), inv, 6144.0) - 6144.0;
                b[i] = (uint32_t)__builtin_bit_cast(uint64_t, r + 6755399441055744.0);
            }
            const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0C0C0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000C0Cu);
            d[j] = (lo | hi) & keep;
        }
        __builtin_memcpy(__builtin_assume_aligned(q + (size_t)c * N, N), d, N);
    };
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = i * TR + t;
        if (c < nvec) put(v[i], c);
    }
    for (int c = NV * TR + t; c < nvec; c += TR) put(load_vec(x, c, K), c);
}

// ----------------------------------------------------------------------------------------------------------- products
//
// y[m][n] = sum_k a[m][k] b[n][k] * sa[m] * sb[n] + bias[n] on v_mfma_i32_16x16x64_i8: weights as the A operand (rows of
// the result tile), tokens as B (columns).  A lane holds 16 codes of a row per multiply; which of a row's codes they are is free as
// long as both operands agree.

template <typename T>
__device__ __forceinline__ void put_result(void* y, int64_t at, float v) {
    static_cast<T*>(y)[at] = (T)v;
}

// a 4 x 4 transpose of bytes: out[o] = byte o of in[0], in[1], in[2], in[3]
__device__ __forceinline__ void transpose_bytes(const uint32_t (&in)[4], uint32_t (&out)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(in[1], in[0], 0x05010400u), b = __builtin_amdgcn_perm(in[1], in[0], 0x07030602u);
    const uint32_t c = __builtin_amdgcn_perm(in[3], in[2], 0x05010400u), d = __builtin_amdgcn_perm(in[3], in[2], 0x07030602u);
    out[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
    out[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
    out[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
    out[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

// 32 lanes of a packed row (bit l: lane l) -> codes: out[o], o < 8, holds lanes o, 8 + o, 16 + o, 24 + o as bytes
template <I8Weights W>
__device__ __forceinline__ void unpack32(uint32_t s, uint32_t z, uint32_t (&out)[8]) {
    if constexpr (W == I8Weights::Ternary) {
        // two bits per lane, sign and zero: even lanes in x, odd ones in y; a byte of 0 .. 3 then picks +1, -1, 0, 0
        const uint32_t x = (s & 0x55555555u) | (z << 1 & 0xAAAAAAAAu), y = (s >> 1 & 0x55555555u) | (z & 0xAAAAAAAAu);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            out[2 * j] = __builtin_amdgcn_perm(0u, 0x0000FF01u, x >> (2 * j) & 0x03030303u);
            out[2 * j + 1] = __builtin_amdgcn_perm(0u, 0x0000FF01u, y >> (2 * j) & 0x03030303u);
        }
    } else {
#pragma unroll
        for (int o = 0; o < 8; o++) out[o] = __builtin_amdgcn_perm(0u, 0x0000FF01u, s >> o & 0x01010101u);
    }
}

// Few tokens: KS wavefronts split K over one tile of 16 weight rows x 16 MB tokens and meet in LDS.
template <I8Weights W, typename T, int MB>
__global__ __launch_bounds__(512) void k_i8_few(I8Product p, uint32_t ntiles) {
    constexpr int KS = 8;
    __shared__ int meet[KS][MB][16][17];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int64_t mt = blockIdx.x / ntiles, n0 = (int64_t)(blockIdx.x - mt * ntiles) * 16, m0 = mt * 16 * MB;
    const int kb = (p.K + 15) & ~15;   // bytes of a row of codes
    v4i acc[MB];
#pragma unroll
    for (int i = 0; i < MB; i++) acc[i] = v4i{0, 0, 0, 0};
    const int8_t* a[MB];
#pragma unroll
    for (int i = 0; i < MB; i++) a[i] = p.a + std::min<int64_t>(m0 + i * 16 + r, p.M - 1) * p.a_stride;
    auto tokens = [&](int i, int k) -> v4i {   // 16 codes from k on; zeros past the row
        return k < kb ? *reinterpret_cast<const v4i*>(a[i] + k) : v4i{0, 0, 0, 0};
    };
    const int64_t n = std::min<int64_t>(n0 + r, p.N - 1);
    if constexpr (W == I8Weights::Codes) {
        const int8_t* const b = static_cast<const int8_t*>(p.b) + n * p.b_stride;
        for (int k0 = wave * 64; k0 < kb; k0 += KS * 64) {
            const int k = k0 + 16 * g;
            const v4i w = k < kb ? *reinterpret_cast<const v4i*>(b + k) : v4i{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < MB; i++) acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w, tokens(i, k), acc[i], 0, 0, 0);
        }
    } else {
        // two groups of four words per step: lane quarter g takes half g % 2 of group g / 2, 128 lanes in 16 bytes of signs (and zeros)
        constexpr bool TERN = W == I8Weights::Ternary;
        const int groups = (p.K + 255) / 256;
        const v4u* const b = static_cast<const v4u*>(p.b) + n * groups * (TERN ? 4 : 2);
        for (int q0 = wave * 2; q0 < groups; q0 += KS * 2) {
            const int q = q0 + (g >> 1), half = g & 1, k0 = q * 256 + half * 128;
            const bool in = q < groups;
            const v4u s = in ? b[q * (TERN ? 4 : 2) + half] : v4u{0, 0, 0, 0}, z = TERN && in ? b[q * 4 + 2 + half] : v4u{0, 0, 0, 0};
#pragma unroll
            for (int d = 0; d < 4; d++) {
                uint32_t w[8];
                unpack32<W>(s[d], z[d], w);
                const v4i w0 = {(int)w[0], (int)w[1], (int)w[2], (int)w[3]}, w1 = {(int)w[4], (int)w[5], (int)w[6], (int)w[7]};
#pragma unroll
                for (int i = 0; i < MB; i++) {
                    const v4i lo = tokens(i, k0 + 32 * d), hi = tokens(i, k0 + 32 * d + 16);
                    uint32_t e[4], o[4];
                    transpose_bytes({(uint32_t)lo[0], (uint32_t)lo[2], (uint32_t)hi[0], (uint32_t)hi[2]}, e);
                    transpose_bytes({(uint32_t)lo[1], (uint32_t)lo[3], (uint32_t)hi[1], (uint32_t)hi[3]}, o);
                    acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w0, v4i{(int)e[0], (int)e[1], (int)e[2], (int)e[3]}, acc[i], 0, 0, 0);
                    acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w1, v4i{(int)o[0], (int)o[1], (int)o[2], (int)o[3]}, acc[i], 0, 0, 0);
                }
            }
        }
    }
    // accumulator e of a lane: weight row 4 g + e, token r
#pragma unroll
    for (int i = 0; i < MB; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) meet[wave][i][r][4 * g + e] = acc[i][e];
    __syncthreads();
    for (int t = threadIdx.x; t < MB * 256; t += 512) {
        const int col = t & 15, tok = t >> 4;
        int sum = 0;
#pragma unroll
        for (int w = 0; w < KS; w++) sum += meet[w][tok >> 4][tok & 15][col];
        const int64_t m = m0 + tok, nn = n0 + col;
        if (m < p.M && nn < p.N) {
            float y = (float)sum * p.sa[m] * p.sb[nn];
            if (p.bias) y += p.bias[nn];
            put_result<T>(p.y, m * p.y_stride + nn, y);
        }
    }
}

}  // namespace

hipError_t launch_quantize_rows_i8(int dtype, const void* d_x, int64_t x_stride, int64_t rows, int K, int8_t* d_q, int64_t q_stride,
                                   float* d_scale, hipStream_t st) {
    return with_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        const T* const x = static_cast<const T*>(d_x);
        k_quantize_rows<T, 4, 1, 4><<<dim3((unsigned)rows), dim3(256), 0, st>>>(x, x_stride, rows, K, d_q, q_stride, d_scale);
        return hipGetLastError();
    });
}

int64_t mm_i8_rows_scratch(I8Weights, int64_t, int64_t, int) { return 0; }

hipError_t launch_mm_i8(I8Weights w, int dtype, const I8Product& p, void*, hipStream_t st) {
    const uint32_t ntiles = (uint32_t)((p.N + 15) / 16);
    auto go = [&](auto weights) {
        constexpr I8Weights W = decltype(weights)::value;
        return with_type(dtype, [&](auto t) {
            typedef decltype(t) T;
            auto run = [&](auto mb) {
                constexpr int MB = decltype(mb)::value;
                const int64_t tiles = ntiles * ((p.M + 16 * MB - 1) / (16 * MB));
                if (tiles > 0x7fffffff) return hipErrorInvalidConfiguration;
                k_i8_few<W, T, MB><<<dim3((unsigned)tiles), dim3(512), 0, st>>>(p, ntiles);
                return hipGetLastError();
            };
            if (p.M <= 16) return run(std::integral_constant<int, 1>{});
            return run(std::integral_constant<int, 2>{});
        });
    };
    if (w == I8Weights::Codes) return go(std::integral_constant<I8Weights, I8Weights::Codes>{});
    if (w == I8Weights::Ternary) return go(std::integral_constant<I8Weights, I8Weights::Ternary>{});
    return go(std::integral_constant<I8Weights, I8Weights::Binary>{});
}

}  // namespace ftnn
