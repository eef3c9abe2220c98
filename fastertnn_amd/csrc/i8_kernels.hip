// Rows of 8-bit codes with a scale each, and their products with 8-bit and with packed ternary or binary weights.
#include <algorithm>

#include "i8_forms.h"
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
// is beyond that is read again, mostly from the L2.  Memory bounds it: 8192 x 11007 float32 109 us, 4.1 TB/s of what has to move (a copy: 5.07).

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

// Few tokens: KS wavefronts split K over one tile of 16 NB weight rows x 16 MB tokens and meet in LDS.  Operands come straight from memory
// into registers, the next step's while this one is multiplied.  What a compute unit can have on its way through its L1 bounds codes (17 bytes per clock; two,
// three or four steps ahead are no faster than one), 1 x 4096 x 4096 6.1 us with its launch; packed weights are bounded by memory for one token (16384 x 16384
// ternary 17.6 us, 3.8 TB/s, from HBM; binary 12.6) and by unpacking, 4 instructions per word of codes, for many.
template <I8Weights W, typename T, int NB, int MB, bool TOKENS>
__global__ __launch_bounds__(512) void k_i8_few(I8Product p, uint32_t ntiles) {
    constexpr int KS = 8, LD = 16 * NB + 4;
    extern __shared__ __align__(16) int meet[];   // [KS][16 MB][LD]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int64_t mt = blockIdx.x / ntiles, n0 = (int64_t)(blockIdx.x - mt * ntiles) * 16 * NB, m0 = mt * 16 * MB;
    const int kb = (p.K + 15) & ~15;   // bytes of a row of codes
    v4i acc[NB][MB];
#pragma unroll
    for (int j = 0; j < NB; j++)
#pragma unroll
        for (int i = 0; i < MB; i++) acc[j][i] = v4i{0, 0, 0, 0};
    const int8_t* a[MB];
#pragma unroll
    for (int i = 0; i < MB; i++) a[i] = p.a + std::min<int64_t>(m0 + i * 16 + r, p.M - 1) * p.a_stride;
    auto piece = [&](const int8_t* row, int k) -> v4i {   // 16 codes from k on; zeros past the row
        return k < kb ? *reinterpret_cast<const v4i*>(row + k) : v4i{0, 0, 0, 0};
    };
    // of a token: none where the lane has no token of its own, which spares the L1 most of the work for one token
    auto token_piece = [&](int i, int k) -> v4i { return k < kb && m0 + 16 * i + r < p.M ? *reinterpret_cast<const v4i*>(a[i] + k) : v4i{0, 0, 0, 0}; };
    if constexpr (W == I8Weights::Codes) {
        const int8_t* b[NB];
#pragma unroll
        for (int j = 0; j < NB; j++) b[j] = static_cast<const int8_t*>(p.b) + std::min<int64_t>(n0 + j * 16 + r, p.N - 1) * p.b_stride;
        // a step is 128 codes of a row, a cache line: two multiplies
        v4i wn[2][NB], tn[2][MB];
        auto fetch = [&](int k0) {
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int k = k0 + 64 * u + 16 * g;
#pragma unroll
                for (int j = 0; j < NB; j++) wn[u][j] = piece(b[j], k);
#pragma unroll
                for (int i = 0; i < MB; i++) tn[u][i] = token_piece(i, k);
            }
        };
        int k0 = wave * 128;
        if (k0 < kb) fetch(k0);
        for (; k0 < kb; k0 += KS * 128) {
            v4i w[2][NB], t[2][MB];
#pragma unroll
            for (int u = 0; u < 2; u++) {
#pragma unroll
                for (int j = 0; j < NB; j++) w[u][j] = wn[u][j];
#pragma unroll
                for (int i = 0; i < MB; i++) t[u][i] = tn[u][i];
            }
            if (k0 + KS * 128 < kb) fetch(k0 + KS * 128);
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int j = 0; j < NB; j++)
#pragma unroll
                    for (int i = 0; i < MB; i++) acc[j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[u][j], t[u][i], acc[j][i], 0, 0, 0);
        }
    } else {
        // two groups of four words per step: lane quarter g takes half g % 2 of group g / 2, 128 lanes in 16 bytes of signs (and zeros)
        constexpr bool TERN = W == I8Weights::Ternary;
        const int groups = (p.K + 255) / 256;
        const v4u* b[NB];
#pragma unroll
        for (int j = 0; j < NB; j++) b[j] = static_cast<const v4u*>(p.b) + std::min<int64_t>(n0 + j * 16 + r, p.N - 1) * groups * (TERN ? 4 : 2);
        // what a step takes: the weights' planes, and of a few tokens (TOKENS) theirs, asked for a step ahead
        static_assert(!TOKENS || MB == 1, "registers for one block of tokens");
        struct Step {
            v4u s[NB], z[NB];
            v4i t[TOKENS ? 8 : 1];
        };
        auto fetch = [&](int q0, Step& x) {
            const int q = q0 + (g >> 1), half = g & 1;
            const bool in = q < groups;
#pragma unroll
            for (int j = 0; j < NB; j++) {
                x.s[j] = in ? b[j][q * (TERN ? 4 : 2) + half] : v4u{0, 0, 0, 0};
                x.z[j] = TERN && in ? b[j][q * 4 + 2 + half] : v4u{0, 0, 0, 0};
            }
            if constexpr (TOKENS) {
#pragma unroll
                for (int d = 0; d < 8; d++) x.t[d] = token_piece(0, q * 256 + half * 128 + 16 * d);
            }
        };
        // word d of quarter g <-> word g of quarter d: then the loads of a word's tokens take 128 codes side by side, whole cache lines, and not 32 each
        // of four (us without / with: 128 x 4096 x 14336 by (4,2) 25.1 / 22.3, 256 x 4096 x 4096 by (4,4) 19.8 / 13.2).  Up to four tokens
        // (TOKENS) have room in the L1 as they are: 1 x 16384 x 16384, weights in the last-level cache, 19.0 / 14.7 without
        auto turn = [&](v4u& w) {
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                const auto s = __builtin_amdgcn_permlane16_swap(w[i], w[i + 1], false, false);
                w[i] = s[0], w[i + 1] = s[1];
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const auto s = __builtin_amdgcn_permlane32_swap(w[i], w[i + 2], false, false);
                w[i] = s[0], w[i + 2] = s[1];
            }
        };
        auto multiply = [&](int q0, Step& x) {
            const int k0 = q0 * 256 + 32 * g;
            if constexpr (!TOKENS) {
#pragma unroll
                for (int j = 0; j < NB; j++) {
                    turn(x.s[j]);
                    if constexpr (TERN) turn(x.z[j]);
                }
            }
#pragma unroll
            for (int d = 0; d < 4; d++) {
                v4i e[MB], o[MB];
#pragma unroll
                for (int i = 0; i < MB; i++) {
                    const v4i lo = TOKENS ? x.t[TOKENS ? 2 * d : 0] : token_piece(i, k0 + 128 * d), hi = TOKENS ? x.t[TOKENS ? 2 * d + 1 : 0] : token_piece(i, k0 + 128 * d + 16);
                    uint32_t u[4], v[4];
                    transpose_bytes({(uint32_t)lo[0], (uint32_t)lo[2], (uint32_t)hi[0], (uint32_t)hi[2]}, u);
                    transpose_bytes({(uint32_t)lo[1], (uint32_t)lo[3], (uint32_t)hi[1], (uint32_t)hi[3]}, v);
                    e[i] = v4i{(int)u[0], (int)u[1], (int)u[2], (int)u[3]}, o[i] = v4i{(int)v[0], (int)v[1], (int)v[2], (int)v[3]};
                }
#pragma unroll
                for (int j = 0; j < NB; j++) {
                    uint32_t w[8];
                    unpack32<W>(x.s[j][d], x.z[j][d], w);
                    const v4i w0 = {(int)w[0], (int)w[1], (int)w[2], (int)w[3]}, w1 = {(int)w[4], (int)w[5], (int)w[6], (int)w[7]};
#pragma unroll
                    for (int i = 0; i < MB; i++) {
                        acc[j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w0, e[i], acc[j][i], 0, 0, 0);
                        acc[j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w1, o[i], acc[j][i], 0, 0, 0);
                    }
                }
            }
        };
        Step now, next;
        int q0 = wave * 2;
        if (q0 < groups) fetch(q0, now);
        for (; q0 < groups; q0 += KS * 4) {   // two steps, so that neither is copied
            if (q0 + KS * 2 < groups) fetch(q0 + KS * 2, next);
            multiply(q0, now);
            if (q0 + KS * 4 < groups) fetch(q0 + KS * 4, now);
            if (q0 + KS * 2 < groups) multiply(q0 + KS * 2, next);
        }
    }
    // accumulator e of a lane: weight row 4 g + e of its block, token r
#pragma unroll
    for (int j = 0; j < NB; j++)
#pragma unroll
        for (int i = 0; i < MB; i++) *reinterpret_cast<v4i*>(meet + (wave * 16 * MB + 16 * i + r) * LD + 16 * j + 4 * g) = acc[j][i];
    __syncthreads();
    for (int t = threadIdx.x; t < 256 * MB * NB; t += 512) {
        const int col = t % (16 * NB), tok = t / (16 * NB);
        int sum = 0;
#pragma unroll
        for (int w = 0; w < KS; w++) sum += meet[(w * 16 * MB + tok) * LD + col];
        const int64_t m = m0 + tok, n = n0 + col;
        if (m < p.M && n < p.N) {
            float y = (float)sum * p.sa[m] * p.sb[n];
            if (p.bias) y += p.bias[n];
            put_result<T>(p.y, m * p.y_stride + n, y);
        }
    }
}

// packed rows -> rows of codes, 32 lanes per thread; stores bound it: 5003 x 4100 in 5 us
template <I8Weights W>
__global__ __launch_bounds__(256) void k_unpack_rows(const uint32_t* __restrict__ B, int64_t N, int K, int8_t* __restrict__ out, int64_t stride) {
    constexpr bool TERN = W == I8Weights::Ternary;
    const int64_t per = stride / 32, words = (int64_t)((K + 255) / 256) * (TERN ? 16 : 8);   // of 32 lanes, of a row
    for (int64_t u = blockIdx.x * 256ll + threadIdx.x; u < N * per; u += gridDim.x * 256ll) {
        const int64_t row = u / per, i = u - row * per;
        const uint32_t* const r = B + row * words + (i / 8) * (TERN ? 16 : 8) + i % 8;
        uint32_t c[8], e[4], o[4];
        unpack32<W>(r[0], TERN ? r[8] : 0u, c);
        transpose_bytes({c[0], c[1], c[2], c[3]}, e);
        transpose_bytes({c[4], c[5], c[6], c[7]}, o);
        v4u* const d = reinterpret_cast<v4u*>(out + row * stride + i * 32);
        d[0] = v4u{e[0], o[0], e[1], o[1]};
        d[1] = v4u{e[2], o[2], e[3], o[3]};
    }
}

}  // namespace

hipError_t launch_quantize_rows_i8(int dtype, const void* d_x, int64_t x_stride, int64_t rows, int K, int8_t* d_q, int64_t q_stride,
                                   float* d_scale, hipStream_t st) {
    return with_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        // A wavefront per row where it holds the row in four vectors a lane (or in one, which leaves more of them at a time), else a workgroup.  us,
        // workgroup / wavefront of four / of one, bf16: 65536 x 128 72.4 / 26.2 / 19.3, 16384 x 512 20.8 / 9.2 / 7.6, 4096 x 2048 9.0 / 7.4 / 7.7,
        // 4096 x 4096 11.4 / 12.4 / 13.1, 8192 x 8192 33.7 / 51.7 / 57.2; few rows alike
        const int nvec = ((K + 15) / 16) * 16 / Vec<T>::N;
        constexpr int64_t kRows = 1 << 23;   // of a launch, which holds fewer than 2^32 threads
        for (int64_t r = 0; r < rows; r += kRows) {
            const int64_t n = std::min(rows - r, kRows);
            const T* const x = static_cast<const T*>(d_x) + r * x_stride;
            const dim3 four((unsigned)((n + 3) / 4));
            if (nvec <= 64) k_quantize_rows<T, 1, 4, 1><<<four, dim3(256), 0, st>>>(x, x_stride, n, K, d_q + r * q_stride, q_stride, d_scale + r);
            else if (nvec <= 256) k_quantize_rows<T, 1, 4, 4><<<four, dim3(256), 0, st>>>(x, x_stride, n, K, d_q + r * q_stride, q_stride, d_scale + r);
            else k_quantize_rows<T, 4, 1, 4><<<dim3((unsigned)n), dim3(256), 0, st>>>(x, x_stride, n, K, d_q + r * q_stride, q_stride, d_scale + r);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
        return hipSuccess;
    });
}

// where packed weights lie as codes: rows of whole cache lines
static int64_t unpacked_stride(int K) { return ((int64_t)K + 127) / 128 * 128; }

// the form without tiles; none (nb 0) where tiles are ahead.  Tiles hold offsets of a row in a tile in 32 bits
static I8Few few_of(I8Weights w, const I8Product& p) {
    const bool packed = w != I8Weights::Codes, wide = p.a_stride >= (8 << 20) || p.b_stride >= (8 << 20);
    const I8Few f = i8_few(packed, p.M, p.N, p.K);
    return f.nb == 0 && wide ? I8Few{1, 2} : f;
}

int64_t mm_i8_rows_scratch(I8Weights w, int64_t M, int64_t N, int K) {
    return i8_few(w != I8Weights::Codes, M, N, K).nb ? 0 : N * unpacked_stride(K);
}

template <I8Weights W>
static hipError_t launch_few(I8Few f, int dtype, const I8Product& p, hipStream_t st) {
    return with_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        auto go = [&](auto nb, auto mb, auto few) {
            constexpr int NB = decltype(nb)::value, MB = decltype(mb)::value, bytes = 8 * 16 * MB * (16 * NB + 4) * 4;
            const int64_t ntiles = (p.N + 16 * NB - 1) / (16 * NB), tiles = ntiles * ((p.M + 16 * MB - 1) / (16 * MB));
            if (tiles >= 1 << 23) return hipErrorInvalidConfiguration;   // a launch holds fewer than 2^32 threads
            auto* const kern = k_i8_few<W, T, NB, MB, decltype(few)::value>;
            static const hipError_t set = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
            if (set != hipSuccess) return set;
            kern<<<dim3((unsigned)tiles), dim3(512), bytes, st>>>(p, (uint32_t)ntiles);
            return hipGetLastError();
        };
        // packed weights: a token's codes are asked for a step ahead up to four tokens; of more they fill the L1.  us, ahead / not, before the turn above: 1 x 16384 x 16384 18.0 / 21.7,
        // 1 x 4096 x 14336 7.0 / 8.5, 16 x 16384 x 16384 26.6 / 23.9, 16 x 4096 x 4096 5.9 / 5.3
        auto run = [&](auto nb, auto mb) {
            if constexpr (W != I8Weights::Codes && decltype(mb)::value == 1)
                if (p.M <= 4) return go(nb, mb, std::true_type{});
            return go(nb, mb, std::false_type{});
        };
        using One = std::integral_constant<int, 1>;
        using Two = std::integral_constant<int, 2>;
        using Four = std::integral_constant<int, 4>;
        if (f.nb == 1 && f.mb == 1) return run(One{}, One{});
        if (f.nb == 2) return run(Two{}, One{});
        if constexpr (W == I8Weights::Codes) {
            return run(One{}, Two{});
        } else {
            if (f.nb == 1) return run(One{}, Two{});   // rows too far apart for tiles
            return f.mb == 1 ? run(Four{}, One{}) : f.mb == 2 ? run(Four{}, Two{}) : run(Four{}, Four{});
        }
    });
}

hipError_t launch_mm_i8(I8Weights w, int dtype, const I8Product& p, void* d_scratch, hipStream_t st) {
    const I8Few f = few_of(w, p);
    if (f.nb) {
        if (w == I8Weights::Codes) return launch_few<I8Weights::Codes>(f, dtype, p, st);
        return w == I8Weights::Ternary ? launch_few<I8Weights::Ternary>(f, dtype, p, st) : launch_few<I8Weights::Binary>(f, dtype, p, st);
    }
    I8Product q = p;
    if (w != I8Weights::Codes) {
        const int64_t stride = unpacked_stride(p.K), units = p.N * (stride / 32);
        auto* const kern = w == I8Weights::Ternary ? k_unpack_rows<I8Weights::Ternary> : k_unpack_rows<I8Weights::Binary>;
        kern<<<dim3((unsigned)std::min<int64_t>((units + 255) / 256, 16384)), dim3(256), 0, st>>>(static_cast<const uint32_t*>(p.b), p.N, p.K, static_cast<int8_t*>(d_scratch), stride);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        q.b = d_scratch, q.b_stride = stride;
    }
    return launch_i8_tiles(dtype, q, st);
}

}  // namespace ftnn
