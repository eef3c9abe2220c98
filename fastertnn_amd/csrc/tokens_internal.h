// Shared by the kernels of token models in few bits (i8_kernels.hip, kv4_kernels.hip) and their C ABI (ftnn_tokens.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/ftnn.h"

namespace ftnn {

int fail(int code, const char* fmt, ...);   // records the text for ftnn_last_error(), returns `code`

// fn(a value of the tensor's element type); dtype is checked before
template <typename F>
auto with_type(int dtype, F&& fn) {
    if (dtype == FTNN_F32) return fn(0.0f);
    if (dtype == FTNN_F16) return fn((_Float16)0.0f);
    return fn((__bf16)0.0f);
}
inline int dtype_bytes(int dtype) { return dtype == FTNN_F32 ? 4 : 2; }

// ---- i8_kernels.hip (arguments already validated) ----
hipError_t launch_quantize_rows_i8(int dtype, const void* d_x, int64_t x_stride, int64_t rows, int K, int8_t* d_q, int64_t q_stride,
                                   float* d_scale, hipStream_t st);

enum class I8Weights { Codes, Ternary, Binary };
struct I8Product {
    const int8_t* a;       // [M] rows of codes, a_stride bytes apart
    int64_t a_stride;
    const float* sa;
    const void* b;         // [N] rows of codes, b_stride bytes apart, or of packed words
    int64_t b_stride;
    const float *sb, *bias;
    int64_t M, N;
    int K;
    void* y;
    int64_t y_stride;
};
hipError_t launch_mm_i8(I8Weights w, int dtype, const I8Product& p, void* d_scratch, hipStream_t st);
// on tiles through LDS (i8_tiles.hip): strides below 8 MiB, weights in codes
hipError_t launch_i8_tiles(int dtype, const I8Product& p, hipStream_t st);
int64_t mm_i8_rows_scratch(I8Weights w, int64_t M, int64_t N, int K);

// ---- kv4_kernels.hip ----
struct Kv4Rotation {
    const float *cos, *sin;
    int positions, rot, neighbours;
};
struct Kv4Rows {   // [tokens][heads][dim], channels contiguous
    const void* p;
    int64_t token_stride, head_stride;
};
hipError_t launch_kv4_append(const ftnn_kv4_t& kv, int dtype, const Kv4Rows& k, const Kv4Rows& v, const Kv4Rotation& r, int heads_q,
                             const Kv4Rows& q, void* d_q_out, hipStream_t st);
hipError_t launch_kv4_read(const ftnn_kv4_t& kv, int dtype, void* d_k, void* d_v, hipStream_t st);
int64_t kv4_attention_scratch(const ftnn_kv4_t& kv, int heads_q, int max_len);
hipError_t launch_kv4_attention(const ftnn_kv4_t& kv, int dtype, int heads_q, const Kv4Rows& q, float scale, int max_len, void* d_out,
                                void* d_scratch, hipStream_t st);

}  // namespace ftnn
