// Products of 8-bit rows with scales on tiles staged through LDS: many tokens.
//
// A workgroup is 2 x 2 wavefronts, each on WN x WM blocks of 32 x 32 (v_mfma_i32_32x32x32_i8): weights as the A operand, so that a lane ends
// with four neighbouring channels of one token in four registers; tokens as B.  A step is 128 codes of every row of the tile: whole cache lines
// (64 codes would fetch every line twice).  They travel global -> LDS by LDS-direct loads of eight rows x 128 bytes, 16
// bytes per lane; the pieces of a row are permuted by its number on the way (piece c of row r lies in place c ^ (r & 7)), so that the 16-byte
// reads of an operand, 32 rows x one piece, spread over all banks.  The loads are counted by hand (s_waitcnt vmcnt); no other
// vector memory is touched before the results, and the launcher refuses a build with scratch memory.
//
// Rows past the operands are clamped (their results are not stored).  A last step of fewer than 128 codes reads its last piece again
// where there are no more, and multiplies only the fragments that hold codes; of the last of those, an upper half without codes is
// cleared in one operand.
//
// The clock under the matrix pipe's load bounds it (1.7 GHz, the pipe busy 68 % of the cycles): 8192 x 8192 x 8192 in 457 us, 2.4 POP/s; smaller ones the rounds of tiles over 256 compute
// units (i8_forms.h).
#include <algorithm>

#include "ftnn_internal.h"
#include "i8_forms.h"
#include "tokens_internal.h"

namespace ftnn {

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));

// M0 carries the LDS address; one wait state after writing it
__device__ __forceinline__ void load_to_lds(uint32_t lds_byte_addr, const int8_t* base, uint32_t offset) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "{m0}"(lds_byte_addr), "v"(offset), "s"(base) : "memory");
}

// Workgroups go to the eight XCDs round-robin; XCD x takes the x-th eighth of the tiles, in bands of four token tiles walked along
// the channels, so that the 32 tiles an XCD works on at a time are about 4 x 8 and share their operands in its L2.
struct TileOrder {
    uint32_t tiles, per_xcd, mt;
    FastDiv band, last;
    __device__ __forceinline__ bool tile(uint32_t wg, int* m, int* n) const {
        const uint32_t t = (wg & 7u) * per_xcd + (wg >> 3);
        if (t >= tiles) return false;
        const uint32_t b = fastdiv(t, band), r = t - b * band.d;
        uint32_t y = r >> 2, x = r & 3u;
        if (b * 4u + 4u > mt) {
            y = fastdiv(r, last);
            x = r - y * last.d;
        }
        *m = (int)(b * 4u + x), *n = (int)y;
        return true;
    }
};

constexpr int BK = 128;   // codes of a step

template <int WM, int WN, int NS, int KG>
struct TileShape {
    static constexpr int RPL = 1024 / BK, PPR = BK / 16;   // rows of a load, pieces of a row
    static constexpr int TM = 64 * WM, TN = 64 * WN, STAGE = (TM + TN) * BK, FM = TM / (4 * RPL), FN = TN / (4 * RPL), FW = FM + FN;
    static __device__ __forceinline__ int swizzle(int r) { return r & (PPR - 1); }
    static constexpr int ring = NS * STAGE, lds = KG * ring + (TM + 2 * TN) * 4;   // a ring per group, and the tile's scales and bias
};

template <typename T, int WM, int WN, int NS, int KG>
__global__ __launch_bounds__(256 * KG) void k_i8_tiles(I8Product p, TileOrder order) {
    typedef TileShape<WM, WN, NS, KG> TS;
    constexpr int TM = TS::TM, TN = TS::TN, FM = TS::FM, FN = TS::FN, FW = TS::FW, NL = WM + WN, NM = WM * WN;
    extern __shared__ __align__(16) int8_t all_lds[];
    const int lane = threadIdx.x & 63, group = KG == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3, wy = wave >> 1, wx = wave & 1;
    int8_t* const lds = all_lds + group * TS::ring;
    const int lr = lane & 31, h = lane >> 5;
    int mt, nt;
    if (!order.tile(blockIdx.x, &mt, &nt)) return;   // (the whole workgroup)
    const int64_t m0 = (int64_t)mt * TM, n0 = (int64_t)nt * TN;
    // whole steps and a last part of one; group g has the steps g, g + KG, ...: `full` whole ones, and the part after them if it is its turn
    const int kb = (p.K + 15) & ~15, whole = kb / BK, full = (whole + KG - 1 - group) / KG, rem = whole % KG == group ? kb % BK : 0, steps = full + (rem != 0);
    const int rounds = (whole + KG - 1) / KG, common = whole / KG;   // of the groups together: every wavefront meets the same barriers

    // load i of a wavefront: eight rows of a side; lane: row lane / 8 of them, piece (lane & 7) ^ (row & 7)
    const int piece = lane % TS::PPR ^ TS::swizzle(lane / TS::PPR);
    uint32_t row_at[FW];
#pragma unroll
    for (int i = 0; i < FW; i++) {
        const int r = TS::RPL * (i < FM ? wave * FM + i : wave * FN + (i - FM)) + lane / TS::PPR;
        row_at[i] = 16u * (uint32_t)piece + (i < FM ? (uint32_t)(std::min<int64_t>(r, p.M - 1 - m0) * p.a_stride) : (uint32_t)(std::min<int64_t>(r, p.N - 1 - n0) * p.b_stride));
    }
    // the tile's scales and bias: fetched ahead of the codes, so that they are there when the sums are
    const float my_sa = p.sa[std::min<int64_t>(m0 + min((int)threadIdx.x, TM - 1), p.M - 1)], my_sb = p.sb[std::min<int64_t>(n0 + min((int)threadIdx.x, TN - 1), p.N - 1)];
    const float my_bias = p.bias ? p.bias[std::min<int64_t>(n0 + min((int)threadIdx.x, TN - 1), p.N - 1)] : 0.0f;
    const int8_t* const a0 = p.a + m0 * p.a_stride;
    const int8_t* const b0 = static_cast<const int8_t*>(p.b) + n0 * p.b_stride;
    const uint32_t lds0 = (uint32_t)(uintptr_t)((__attribute__((address_space(3))) void*)all_lds) + (uint32_t)(group * TS::ring);
    auto load = [&](int step, int i, auto all) {   // all: of the step's codes exist
        constexpr bool WHOLE = decltype(all)::value;
        const uint32_t dst = lds0 + (uint32_t)(step % NS) * TS::STAGE + (i < FM ? (uint32_t)(wave * FM + i) : (uint32_t)(TM / TS::RPL + wave * FN + (i - FM))) * 1024u;
        const uint32_t back = WHOLE || step < full ? 0u : 16u * (uint32_t)max(piece - (rem / 16 - 1), 0);   // the last piece again
        load_to_lds(dst, (i < FM ? a0 : b0) + ((int64_t)step * KG + group) * BK, row_at[i] - back);
    };
    // operand block j of a side, fragment k (32 codes) of a step
    auto tokens = [&](int step, int k, int j) -> v4i {
        const int r = (wy * WM + j) * 32 + lr;
        return *reinterpret_cast<const v4i*>(lds + (step % NS) * TS::STAGE + r * BK + ((2 * k + h) ^ TS::swizzle(r)) * 16);
    };
    auto weights = [&](int step, int k, int j) -> v4i {
        const int r = (wx * WN + j) * 32 + lr;
        return *reinterpret_cast<const v4i*>(lds + (step % NS) * TS::STAGE + TM * BK + r * BK + ((2 * k + h) ^ TS::swizzle(r)) * 16);
    };
    v16i acc[WN][WM];
#pragma unroll
    for (int a = 0; a < WN; a++)
#pragma unroll
        for (int b = 0; b < WM; b++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[a][b][e] = 0;
    v4i fw[2][WN], ft[2][WM];
    auto read = [&](int step, int k, int set, int i) {   // in the order in which the multiplies take them
        if (i == 0) fw[set][0] = weights(step, k, 0);
        else if (i <= WM) ft[set][i - 1] = tokens(step, k, i - 1);
        else fw[set][i - WM] = weights(step, k, i - WM);
    };
    auto multiply = [&](int set, int i) {   // those that go with read i
#pragma unroll
        for (int m = i * NM / NL; m < (i + 1) * NM / NL; m++)
            acc[m / WM][m % WM] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[set][m / WM], ft[set][m % WM], acc[m / WM][m % WM], 0, 0, 0);
    };

#pragma unroll
    for (int s = 0; s < NS; s++)
        if (s < steps) {
#pragma unroll
            for (int i = 0; i < FW; i++) load(s, i, std::false_type{});
        }
    if (steps >= NS) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(FW * (NS - 1)) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (full > 0) {
#pragma unroll
        for (int i = 0; i < NL; i++) read(0, 0, 0, i);
    }
    // BUSY: steps s + 1 .. s + NS are whole ones
    auto step_of = [&](int s, auto busy) {
        constexpr bool BUSY = decltype(busy)::value;
        const bool mine = BUSY || KG == 1 || s < full;   // (a group with a step less meets the barriers)
#pragma unroll
        for (int k = 0; k < BK / 32; k++) {
            const int set = k & 1;
            if (k < BK / 32 - 1) {
#pragma unroll
                for (int i = 0; i < NL; i++) {
                    if (mine) {
                        read(s, k + 1, set ^ 1, i);
                        multiply(set, i);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            } else {
                // all of this step is in registers; step s + 1 has to have landed, steps s + 2 .. s + NS - 1 may be in flight; behind the barrier
                // this step's place is free for step s + NS
                if (BUSY || s + NS - 1 < steps) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(FW * (NS - 2)) : "memory");
                else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads();
                const bool more = BUSY || s + NS < steps, next = BUSY || s + 1 < full;
#pragma unroll
                for (int i = 0; i < NL; i++) {
                    if (more) {
#pragma unroll
                        for (int j = i * FW / NL; j < (i + 1) * FW / NL; j++) load(s + NS, j, busy);
                    }
                    if (next) read(s + 1, 0, set ^ 1, i);
                    if (mine) multiply(set, i);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
    };
    int s = 0;
    for (; s + NS < common; s++) step_of(s, std::true_type{});
    for (; s < rounds; s++) step_of(s, std::false_type{});
    if (rem) {
        for (int k = 0; 32 * k < rem; k++) {
#pragma unroll
            for (int i = 0; i < NL; i++) read(full, k, 0, i);
            const int keep = 32 * k + 16 * h < rem ? -1 : 0;
#pragma unroll
            for (int b = 0; b < WM; b++) ft[0][b] &= keep;
#pragma unroll
            for (int i = 0; i < NL; i++) multiply(0, i);
        }
    }
    if constexpr (KG > 1) {   // the groups' sums meet in the first one
        static_assert((KG - 1) * NM * 16 * 256 * 4 <= KG * TS::ring, "the sums fit the rings");
        __syncthreads();
        if (group) {
#pragma unroll
            for (int m = 0; m < NM; m++) {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    *reinterpret_cast<v4i*>(all_lds + ((((group - 1) * NM + m) * 4 + e) * 256 + (int)(threadIdx.x & 255)) * 16) =
                        v4i{acc[m / WM][m % WM][4 * e], acc[m / WM][m % WM][4 * e + 1], acc[m / WM][m % WM][4 * e + 2], acc[m / WM][m % WM][4 * e + 3]};
            }
        }
        __syncthreads();
        if (group) return;   // (nothing below waits for these wavefronts: a barrier counts those that are left)
#pragma unroll
        for (int o = 0; o < (KG - 1) * NM; o++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const v4i v = *reinterpret_cast<const v4i*>(all_lds + ((o * 4 + e) * 256 + (int)threadIdx.x) * 16);
#pragma unroll
                for (int x = 0; x < 4; x++) acc[o % NM / WM][o % NM % WM][4 * e + x] += v[x];
            }
    }
    // Results leave through LDS, 32 tokens at a time, so that a row's channels are stored in pieces of 16 bytes side by side.  Accumulator e of block
    // (a, b): channel 32 a + 8 (e / 4) + 4 h + e % 4, token 32 b + lr.
    constexpr int PITCH = 32 * WN * (int)sizeof(T) + 16, EV = 16 / (int)sizeof(T), PIECES = 32 * WN / EV, ROWS = 64 / PIECES;   // rows per store
    static_assert(4 * 32 * PITCH <= TS::ring, "the results' rows fit the ring");
    static_assert(64 % PIECES == 0, "whole rows per store");
    float* const scales = reinterpret_cast<float*>(all_lds + KG * TS::ring);   // of the tokens, of the channels, bias
    if (threadIdx.x < TM) scales[threadIdx.x] = my_sa;
    if (threadIdx.x < TN) scales[TM + threadIdx.x] = my_sb, scales[TM + TN + threadIdx.x] = my_bias;
    __syncthreads();   // and no wavefront reads the ring any more
    int8_t* const mine = lds + wave * 32 * PITCH;
    const int64_t nw = n0 + wx * WN * 32, mw = m0 + wy * WM * 32;
#pragma unroll
    for (int b = 0; b < WM; b++) {
        const float sa = scales[(wy * WM + b) * 32 + lr];
#pragma unroll
        for (int a = 0; a < WN; a++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float* const at = scales + TM + (wx * WN + a) * 32 + 8 * e + 4 * h;
                const float4 sb = *reinterpret_cast<const float4*>(at), c = *reinterpret_cast<const float4*>(at + TN);
                // (adding 0 where there is no bias makes +0 of a sum of -0, which no sum of whole numbers is)
                const float4 y = make_float4((float)acc[a][b][4 * e] * sa * sb.x + c.x, (float)acc[a][b][4 * e + 1] * sa * sb.y + c.y,
                                             (float)acc[a][b][4 * e + 2] * sa * sb.z + c.z, (float)acc[a][b][4 * e + 3] * sa * sb.w + c.w);
                const T r[4] = {(T)y.x, (T)y.y, (T)y.z, (T)y.w};
                __builtin_memcpy(__builtin_assume_aligned(mine + lr * PITCH + (32 * a + 8 * e + 4 * h) * sizeof(T), sizeof(r)), r, sizeof(r));
            }
#pragma unroll
        for (int i = 0; i < 32 / ROWS; i++) {
            const int r = i * ROWS + lane / PIECES, c = lane % PIECES;
            const v4i v = *reinterpret_cast<const v4i*>(mine + r * PITCH + c * 16);
            const int64_t m = mw + 32 * b + r, n = nw + c * EV;
            if (m < p.M) {
                T* const y = static_cast<T*>(p.y) + m * p.y_stride + n;   // rows may start at any value
                if (n + EV <= p.N) {
                    __builtin_memcpy(y, &v, 16);
                } else {
                    T x[EV];
                    __builtin_memcpy(x, &v, 16);
#pragma unroll
                    for (int j = 0; j < EV; j++)
                        if (n + j < p.N) y[j] = x[j];
                }
            }
        }
    }
}

template <typename T, int WM, int WN, int NS, int KG>
hipError_t launch(const I8Product& p, hipStream_t st) {
    typedef TileShape<WM, WN, NS, KG> TS;
    auto* const kern = k_i8_tiles<T, WM, WN, NS, KG>;
    static const hipError_t configured = [&]() {
        hipFuncAttributes attr;   // a scratch access would move the count that the waits rely on
        hipError_t e = hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(kern));
        if (e == hipSuccess && attr.localSizeBytes != 0) e = hipErrorLaunchFailure;
        if (e != hipSuccess) return e;
        return hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, TS::lds);
    }();
    if (configured != hipSuccess) return configured;
    const int64_t mt = (p.M + TS::TM - 1) / TS::TM, nt = (p.N + TS::TN - 1) / TS::TN;
    if (mt * nt >= (1 << 24) / KG - 8) return hipErrorInvalidConfiguration;   // a launch holds fewer than 2^32 threads
    TileOrder o;
    o.tiles = (uint32_t)(mt * nt), o.per_xcd = (o.tiles + 7) / 8, o.mt = (uint32_t)mt;
    o.band = make_fastdiv((uint32_t)(4 * nt)), o.last = make_fastdiv((uint32_t)(mt % 4 ? mt % 4 : 4));
    hipLaunchKernelGGL(kern, dim3(8 * o.per_xcd), dim3(256 * KG), TS::lds, st, p, o);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_i8_tiles(int dtype, const I8Product& p, hipStream_t st) {
    return with_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        switch (i8_form(p.M, p.N, p.K)) {
            case I8Form::T256: return launch<T, 4, 4, 2, 1>(p, st);
            case I8Form::T128: return launch<T, 2, 2, 4, 1>(p, st);
            case I8Form::T128Two: return launch<T, 2, 2, 2, 1>(p, st);
            case I8Form::T128x64: return launch<T, 2, 1, 3, 1>(p, st);
            case I8Form::T64: return launch<T, 1, 1, 4, 1>(p, st);
            default: return launch<T, 1, 1, 4, 2>(p, st);
        }
    });
}

}  // namespace ftnn
