// C ABI of the operators of token models in few bits: argument checking (include/ftnn.h, part 3).
#include <math.h>

#include "tokens_internal.h"

using namespace ftnn;

namespace {

constexpr int kMaxCodes = 131071;   // K * 128 * 128 below 2^31

bool aligned(const void* p, int to) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(to - 1)) == 0; }

int done(hipError_t e, const char* what) {
    return e == hipSuccess ? FTNN_OK : fail(FTNN_EHIP, "%s: %s", what, hipGetErrorString(e));
}

int check_type(int dtype) {
    return dtype == FTNN_F32 || dtype == FTNN_F16 || dtype == FTNN_BF16 ? FTNN_OK : fail(FTNN_EINVAL, "unknown element type %d", dtype);
}

int check_product(int dtype, const I8Product& p) {
    if (const int rc = check_type(dtype)) return rc;
    if (p.M < 0 || p.N <= 0 || p.K <= 0) return fail(FTNN_EINVAL, "non-positive dimension");
    if (p.K > kMaxCodes) return fail(FTNN_EINVAL, "rows of %d codes: 32-bit sums hold %d", p.K, kMaxCodes);
    if (p.M > INT32_MAX || p.N > INT32_MAX || p.M * p.N >= (int64_t)1 << 40) return fail(FTNN_EINVAL, "more than 2^31 - 1 rows or 2^40 results");
    if (p.M == 0) return FTNN_OK;
    if (!p.a || !p.sa || !p.b || !p.sb || !p.y) return fail(FTNN_EINVAL, "null pointer");
    if (!aligned(p.a, 16) || !aligned(p.b, 16)) return fail(FTNN_EINVAL, "operands must be 16-byte aligned");
    if (!aligned(p.sa, 4) || !aligned(p.sb, 4) || !aligned(p.bias, 4) || !aligned(p.y, dtype_bytes(dtype)))
        return fail(FTNN_EINVAL, "scales, bias and result must be aligned to their type");
    if (p.a_stride % 16 || p.a_stride < ftnn_i8_row_bytes(p.K)) return fail(FTNN_EINVAL, "rows of codes must be a multiple of 16 bytes apart, %lld at least", (long long)ftnn_i8_row_bytes(p.K));
    if (p.y_stride < p.N) return fail(FTNN_EINVAL, "result rows overlap");
    return FTNN_OK;
}

int check_kv(const ftnn_kv4_t* kv) {
    if (!kv) return fail(FTNN_EINVAL, "null pointer");
    if (kv->heads <= 0 || ftnn_kv4_page_bytes(kv->heads, kv->dim, kv->page) < 0)
        return fail(FTNN_EINVAL, "heads %d, dim %d, page %d: dim is 64, 96, 128 or 256, page 16, 32, 64, 128 or 256", kv->heads, kv->dim, kv->page);
    if (kv->sequences < 0 || kv->tokens < 0 || kv->width <= 0 || kv->pages <= 0 || kv->pages > INT32_MAX) return fail(FTNN_EINVAL, "non-positive dimension");
    if ((int64_t)kv->width * kv->page > 1 << 30) return fail(FTNN_EINVAL, "sequences of more than 2^30 tokens");
    if (kv->heads > 32767) return fail(FTNN_EINVAL, "more than 32767 heads");
    if (kv->table_stride < kv->width) return fail(FTNN_EINVAL, "rows of the table overlap");
    if (!kv->tokens || !kv->sequences) return FTNN_OK;
    if (!kv->d_cache || !kv->d_table || !kv->d_lens || !kv->d_starts) return fail(FTNN_EINVAL, "null pointer");
    if (!aligned(kv->d_cache, 16)) return fail(FTNN_EINVAL, "the cache must be 16-byte aligned");
    if (!aligned(kv->d_table, 4) || !aligned(kv->d_lens, 4) || !aligned(kv->d_starts, 4)) return fail(FTNN_EINVAL, "table, lens and starts must be aligned to their type");
    return FTNN_OK;
}

int check_heads_q(const ftnn_kv4_t* kv, int heads_q) {
    if (heads_q <= 0 || heads_q % kv->heads) return fail(FTNN_EINVAL, "%d query heads over %d heads", heads_q, kv->heads);
    if (heads_q > 32767 || (int64_t)kv->tokens * heads_q > INT32_MAX) return fail(FTNN_EINVAL, "more than 2^31 - 1 query rows, or 32767 heads");
    return FTNN_OK;
}

int mm_i8(I8Weights w, int dtype, const I8Product& p, void* d_scratch, int64_t scratch_bytes, int64_t need, void* stream) {
    if (const int rc = check_product(dtype, p)) return rc;
    if (p.M == 0) return FTNN_OK;
    if (need > 0 && (!d_scratch || scratch_bytes < need || !aligned(d_scratch, 16)))
        return fail(FTNN_EINVAL, "scratch must be 16-byte aligned and hold %lld bytes", (long long)need);
    return done(launch_mm_i8(w, dtype, p, d_scratch, static_cast<hipStream_t>(stream)), "8-bit product");
}

}  // namespace

extern "C" {

int64_t ftnn_i8_row_bytes(int K) { return ((int64_t)K + 15) / 16 * 16; }

int ftnn_quantize_rows_i8(int dtype, const void* d_x, int64_t x_stride, int64_t rows, int K, int8_t* d_q, int64_t q_stride, float* d_scale,
                          void* stream) {
    if (const int rc = check_type(dtype)) return rc;
    if (rows < 0 || rows > INT32_MAX || K <= 0) return fail(FTNN_EINVAL, "%lld rows of %d values", (long long)rows, K);
    if (K > INT32_MAX - 65536) return fail(FTNN_EINVAL, "rows of more than %d values", INT32_MAX - 65536);
    if (rows == 0) return FTNN_OK;
    if (!d_x || !d_q || !d_scale) return fail(FTNN_EINVAL, "null pointer");
    if (!aligned(d_x, dtype_bytes(dtype)) || !aligned(d_scale, 4) || !aligned(d_q, 16)) return fail(FTNN_EINVAL, "codes must be 16-byte aligned, values and scales to their type");
    if (q_stride % 16 || q_stride < ftnn_i8_row_bytes(K)) return fail(FTNN_EINVAL, "rows of codes must be a multiple of 16 bytes apart, %lld at least", (long long)ftnn_i8_row_bytes(K));
    if (x_stride < 0) return fail(FTNN_EINVAL, "negative stride");
    return done(launch_quantize_rows_i8(dtype, d_x, x_stride, rows, K, d_q, q_stride, d_scale, static_cast<hipStream_t>(stream)), "rows to 8-bit codes");
}

int ftnn_mm_i8(int dtype, const int8_t* d_a, int64_t a_stride, const float* d_sa, const int8_t* d_b, int64_t b_stride, const float* d_sb,
               const float* d_bias, int64_t M, int64_t N, int K, void* d_y, int64_t y_stride, void* stream) {
    if (K > 0 && (b_stride % 16 || b_stride < ftnn_i8_row_bytes(K)))
        return fail(FTNN_EINVAL, "rows of codes must be a multiple of 16 bytes apart, %lld at least", (long long)ftnn_i8_row_bytes(K));
    return mm_i8(I8Weights::Codes, dtype, {d_a, a_stride, d_sa, d_b, b_stride, d_sb, d_bias, M, N, K, d_y, y_stride}, nullptr, 0, 0, stream);
}

int64_t ftnn_mm_i8_rows_scratch_bytes(int ternary, int64_t M, int64_t N, int K) {
    if (M <= 0 || N <= 0 || K <= 0 || K > kMaxCodes) return 0;
    return mm_i8_rows_scratch(ternary ? I8Weights::Ternary : I8Weights::Binary, M, N, K);
}

int ftnn_mm_i8_rows(int ternary, int dtype, const int8_t* d_a, int64_t a_stride, const float* d_sa, const int64_t* d_b, const float* d_sb,
                    const float* d_bias, int64_t M, int64_t N, int K, void* d_y, int64_t y_stride, void* d_scratch, int64_t scratch_bytes,
                    void* stream) {
    return mm_i8(ternary ? I8Weights::Ternary : I8Weights::Binary, dtype, {d_a, a_stride, d_sa, d_b, 0, d_sb, d_bias, M, N, K, d_y, y_stride}, d_scratch,
                 scratch_bytes, ftnn_mm_i8_rows_scratch_bytes(ternary, M, N, K), stream);
}

int64_t ftnn_kv4_page_bytes(int heads, int dim, int page) {
    if (heads <= 0) return fail(FTNN_EINVAL, "%d heads", heads);
    if (dim != 64 && dim != 96 && dim != 128 && dim != 256) return fail(FTNN_EINVAL, "heads of %d channels: 64, 96, 128 or 256", dim);
    if (page < 16 || page > 256 || (page & (page - 1))) return fail(FTNN_EINVAL, "pages of %d tokens: 16, 32, 64, 128 or 256", page);
    return (int64_t)heads * page * (dim + 8);
}

int ftnn_kv4_append(const ftnn_kv4_t* kv, int dtype, const void* d_k, int64_t k_token_stride, int64_t k_head_stride, const void* d_v,
                    int64_t v_token_stride, int64_t v_head_stride, const float* d_cos, const float* d_sin, int positions, int rot, int neighbours,
                    int heads_q, const void* d_q, int64_t q_token_stride, int64_t q_head_stride, void* d_q_out, void* stream) {
    if (const int rc = check_type(dtype)) return rc;
    if (const int rc = check_kv(kv)) return rc;
    if (heads_q < 0 || heads_q > 32767) return fail(FTNN_EINVAL, "%d query heads", heads_q);
    if (rot < 0 || rot > kv->dim || rot % 2) return fail(FTNN_EINVAL, "rotation of %d of %d channels", rot, kv->dim);
    if (rot && (positions < 0 || ((!d_cos || !d_sin) && positions > 0) || !aligned(d_cos, 4) || !aligned(d_sin, 4))) return fail(FTNN_EINVAL, "rotation without tables");
    if (!kv->tokens || !kv->sequences) return FTNN_OK;
    const int size = dtype_bytes(dtype);
    if (!d_k || !d_v || (heads_q && (!d_q || !d_q_out))) return fail(FTNN_EINVAL, "null pointer");
    if (!aligned(d_k, size) || !aligned(d_v, size) || !aligned(d_q, size) || !aligned(d_q_out, size)) return fail(FTNN_EINVAL, "tensors must be aligned to their type");
    return done(launch_kv4_append(*kv, dtype, {d_k, k_token_stride, k_head_stride}, {d_v, v_token_stride, v_head_stride},
                                  {d_cos, d_sin, positions, rot, neighbours != 0}, heads_q, {d_q, q_token_stride, q_head_stride}, d_q_out,
                                  static_cast<hipStream_t>(stream)), "append to the cache");
}

int ftnn_kv4_read(const ftnn_kv4_t* kv, int dtype, void* d_k, void* d_v, void* stream) {
    if (const int rc = check_type(dtype)) return rc;
    if (const int rc = check_kv(kv)) return rc;
    if (!kv->tokens || !kv->sequences || (!d_k && !d_v)) return FTNN_OK;
    if (!aligned(d_k, dtype_bytes(dtype)) || !aligned(d_v, dtype_bytes(dtype))) return fail(FTNN_EINVAL, "tensors must be aligned to their type");
    return done(launch_kv4_read(*kv, dtype, d_k, d_v, static_cast<hipStream_t>(stream)), "read from the cache");
}

int64_t ftnn_kv4_attention_scratch_bytes(const ftnn_kv4_t* kv, int heads_q, int max_len) {
    if (!kv || kv->heads <= 0 || kv->tokens <= 0 || kv->sequences <= 0 || kv->width <= 0 || kv->page <= 0 || heads_q < kv->heads || heads_q % kv->heads) return 0;
    return kv4_attention_scratch(*kv, heads_q, max_len);
}

int ftnn_kv4_attention(const ftnn_kv4_t* kv, int dtype, int heads_q, const void* d_q, int64_t q_token_stride, int64_t q_head_stride, float scale,
                       int max_len, void* d_out, void* d_scratch, int64_t scratch_bytes, void* stream) {
    if (dtype != FTNN_F16 && dtype != FTNN_BF16) return fail(FTNN_EINVAL, "attention takes FTNN_F16 and FTNN_BF16");
    if (const int rc = check_kv(kv)) return rc;
    if (const int rc = check_heads_q(kv, heads_q)) return rc;
    if (!(scale > 0.0f) || !(scale < INFINITY)) return fail(FTNN_EINVAL, "scale has to be positive and finite");
    if (max_len < 0) return fail(FTNN_EINVAL, "max_len %d", max_len);
    if (!kv->tokens || !kv->sequences) return FTNN_OK;
    if (!d_q || !d_out) return fail(FTNN_EINVAL, "null pointer");
    if (!aligned(d_q, 2) || !aligned(d_out, 2)) return fail(FTNN_EINVAL, "tensors must be aligned to their type");
    const int64_t need = kv4_attention_scratch(*kv, heads_q, max_len);
    if (need > 0 && (!d_scratch || scratch_bytes < need || !aligned(d_scratch, 16)))
        return fail(FTNN_EINVAL, "scratch must be 16-byte aligned and hold %lld bytes", (long long)need);
    return done(launch_kv4_attention(*kv, dtype, heads_q, {d_q, q_token_stride, q_head_stride}, scale, max_len, d_out, d_scratch,
                                     static_cast<hipStream_t>(stream)), "attention");
}

}  // extern "C"
