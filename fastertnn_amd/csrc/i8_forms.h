// Which form a product of 8-bit rows takes (host code; run on the CPU by tests/test_i8_forms.py).
#pragma once
#include <stdint.h>

namespace ftnn {

// Tiles of tokens x channels: one workgroup of 4 wavefronts per compute unit with a deep ring, or two with a shallow one (T128Two); T64Split:
// 8 wavefronts, two groups of 4 that split K.
enum class I8Form { T256, T128, T128Two, T128x64, T64, T64Split };

// Microseconds of 128 codes of K, as measured with the chip full (K from 512 to 14336; a launch is 4 us on top): `one` where a compute
// unit has one workgroup, `two` where it has two.  256 x 256: 4096 x 4096 x 4096 65 us, 8192 x 8192 x 8192 454.  128 x 128: 1024 x 4096 x 4096 22.4
// (deep ring; 25.2 shallow), 2048 x 4096 x 4096 38.7 (shallow, two per unit; 43.0 deep).  128 x 64: 512 x 4096 x 4096 16.3 (64 x 64: 18.4).  64 x 64:
// 256 x 4096 x 4096 11.3 (128 x 128: 18.0); 64 x 4096 x 14336 26.0, with K split 22.8.
inline double i8_rounds(int64_t tiles, double one, double two) {
    const int64_t rest = tiles % 512;
    return (double)(tiles / 512) * two + (rest == 0 ? 0.0 : rest <= 256 ? one : two);
}
struct I8Estimate {
    I8Form form;
    double us;   // of 128 codes of K
};
inline I8Estimate i8_estimate(int64_t M, int64_t N, int K) {
    auto tiles = [&](int64_t m, int64_t n) { return ((M + m - 1) / m) * ((N + n - 1) / n); };
    const int64_t t128 = tiles(128, 128), t64 = tiles(64, 64);
    const double e256 = 1.8 * (double)((tiles(256, 256) + 255) / 256), e128 = i8_rounds(t128, 0.55, 1.08);
    const double e12864 = i8_rounds(tiles(128, 64), 0.38, 0.68), e64 = i8_rounds(t64, 0.2, 0.45);
    if (e64 <= e12864 && e64 <= e128 && e64 <= e256) return {t64 <= 256 && K >= 8192 ? I8Form::T64Split : I8Form::T64, e64};
    if (e12864 <= e128 && e12864 <= e256) return {I8Form::T128x64, e12864};
    if (e128 <= e256) return {t128 <= 256 ? I8Form::T128 : I8Form::T128Two, e128};
    return {I8Form::T256, e256};
}
inline I8Form i8_form(int64_t M, int64_t N, int K) { return i8_estimate(M, N, K).form; }

// Few tokens run without tiles: workgroups of 8 wavefronts that split K over nb x 16 channels and mb x 16 tokens (nb 0: tiles).  For codes, and packed
// weights under up to 16 tokens or a chipful of the smallest workgroups, the form is the first of a list with about one workgroup per compute unit or
// fewer: the smaller ones spread the work, the larger ones read less of the other operand again.  Codes, us: 1 x 4096 x 4096 (1,1) 6.1, (2,1) 6.6,
// tiles 9.9; 1 x 8192 x 4096 10.5, 8.8, 9.9; 1 x 14336 x 4096 14.9, 12.7, 11.3; 32 x 4096 x 4096 (1,1) 10.3, (1,2) 8.3, tiles 9.9;
// 64 x 1024 x 1024 (1,1) 3.7, tiles 5.2; 64 x 4096 x 4096 (2,2) 10.1, tiles 10.1.  Packed weights: 16 x 16384 x 16384 (1,1) 40.5, (4,1) 23.5.
//
// More tokens over packed weights go by an estimate: microseconds of 128 codes of K for a round of 256 workgroups, and for tiles those above with the
// launch that unpacks the weights (4 us and 0.18 for a million codes).  us, (4,1), (4,2), (4,4), tiles: 64 x 4096 x 4096 7.4, 8.7, 12.6, 24.4;
// 256 x 4096 x 4096 20.0, 16.1, 13.2, 25.5; 512 x 1024 x 4096 11.4, 8.6, 12.8, 15.7; 117 x 9054 x 10539 54, 54, 48, 57; 128 x 14336 x 4096 33.2, 30.5, 24.8, 37.0;
// 256 x 8192 x 8192 68.7, 52.7, 42.7, 47.2; 512 x 4096 x 4096 36.8, 30.4, 24.2, 28.7; 2269 x 4910 x 420 81.9, 94.9, 69.9, 21.6.
struct I8Few {
    int nb, mb;
};
inline I8Few i8_few(bool packed, int64_t M, int64_t N, int K) {
    auto workgroups = [&](int nb, int mb) { return ((N + 16 * nb - 1) / (16 * nb)) * ((M + 16 * mb - 1) / (16 * mb)); };
    auto fits = [&](int nb, int mb) { return workgroups(nb, mb) <= 320; };
    if (fits(1, 1)) return {1, 1};
    if (!packed) {
        if (M > 16) return fits(1, 2) ? I8Few{1, 2} : I8Few{0, 0};
        return fits(2, 1) ? I8Few{2, 1} : I8Few{0, 0};
    }
    if (fits(2, 1)) return {2, 1};
    if (M <= 16) return {4, 1};
    I8Few best = {0, 0};
    double least = i8_estimate(M, N, K).us + 4.0 * 128 / K + 0.18e-6 * 128 * (double)N;
    auto consider = [&](int mb, double one) {
        const double us = one * (double)((workgroups(4, mb) + 255) / 256);
        if (us < least) best = {4, mb}, least = us;
    };
    consider(1, 0.11), consider(2, 0.16), consider(4, 0.27);
    return best;
}

}  // namespace ftnn
