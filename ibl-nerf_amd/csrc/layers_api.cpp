// C entries of the trainable-layer operators (include/iblnerf_layers.h): argument checks, then launches.  No state: every buffer is the caller's.
#include <cstdarg>
#include <cstdio>

#include "../../include/iblnerf_layers.h"
#include "layers.h"

using namespace ibl;

namespace {

thread_local char g_error[512] = "";

int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_error, sizeof g_error, fmt, ap);
    va_end(ap);
    return code;
}

int done(const char* who, hipError_t e) { return e == hipSuccess ? IBLNERF_OK : fail(IBLNERF_ERR_HIP, "%s: %s", who, hipGetErrorString(e)); }

constexpr int64_t MAX_ROWS = INT32_MAX - 1023;
constexpr int MAX_COLS = 65536;

bool bad_type(int t) { return t < IBLNERF_FLOAT32 || t > IBLNERF_FLOAT16; }
constexpr int64_t MAX_STRIDE = 1 << 24;      // (a tile's rows are reached by 32-bit offsets)
// rows [n][cols] at p: enough stride, a pointer where there is something, aligned to the element
bool bad_rows(const void* p, int64_t ld, int64_t n, int64_t cols, int dtype) {
    return n > 0 && (!p || ld < cols || ld > MAX_STRIDE || (reinterpret_cast<uintptr_t>(p) & (dtype == IBLNERF_FLOAT32 ? 3 : 1)) != 0);
}
bool bad_codes(const void* p) { return !p || (reinterpret_cast<uintptr_t>(p) & 7) != 0; }
bool bad_workspace(const void* p, size_t bytes, size_t need) { return need > 0 && (!p || bytes < need || (reinterpret_cast<uintptr_t>(p) & 15) != 0); }
// a launch holds fewer than 2^32 threads
bool too_many_tiles(int64_t n, int o) { return (n / 128 + 9) * (int64_t)((o + 127) / 128) >= (1 << 24); }

}  // namespace

extern "C" {

const char* iblnerf_layers_last_error(void) { return g_error; }

int iblnerf_checkpoint(void* stream, int dtype, const void* d_x, int64_t ld_x, int64_t n, int k, int is_signed, uint8_t* d_codes, uint8_t* d_scales) {
    if (bad_type(dtype) || n < 0 || n > MAX_ROWS || k < 1 || k > MAX_COLS || bad_rows(d_x, ld_x, n, k, dtype) || (n > 0 && (bad_codes(d_codes) || !d_scales)))
        return fail(IBLNERF_ERR_INVALID, "checkpoint: bad arguments (dtype %d, n=%lld, k=%d, ld=%lld)", dtype, (long long)n, k, (long long)ld_x);
    if (n == 0) return IBLNERF_OK;
    return done("checkpoint", launch_checkpoint(dtype, d_x, ld_x, n, k, is_signed != 0, d_codes, d_scales, (hipStream_t)stream));
}

int iblnerf_checkpoint_values(void* stream, const uint8_t* d_codes, const uint8_t* d_scales, int64_t n, int k, int is_signed, int dtype, void* d_out, int64_t ld_out) {
    if (bad_type(dtype) || n < 0 || n > MAX_ROWS || k < 1 || k > MAX_COLS || bad_rows(d_out, ld_out, n, k, dtype) || (n > 0 && (bad_codes(d_codes) || !d_scales)))
        return fail(IBLNERF_ERR_INVALID, "checkpoint_values: bad arguments (dtype %d, n=%lld, k=%d, ld=%lld)", dtype, (long long)n, k, (long long)ld_out);
    if (n == 0) return IBLNERF_OK;
    return done("checkpoint_values", launch_checkpoint_values(dtype, Checkpoint8{d_codes, d_scales, is_signed != 0}, n, k, d_out, ld_out, (hipStream_t)stream));
}

size_t iblnerf_dense_forward_workspace(int dtype, int64_t n, int k, int o) {
    if (bad_type(dtype) || n < 0 || n > MAX_ROWS || k < 1 || k > MAX_COLS || o < 1 || o > MAX_COLS) return 0;
    return dense_rows_bytes(dtype, n, k, o);
}

int iblnerf_dense_forward(void* stream, int dtype, const void* d_x, int64_t ld_x, int64_t n, int k, const void* d_w, int64_t ld_w, int o, const void* d_bias, int relu,
                          void* d_y, int64_t ld_y, uint8_t* d_codes, uint8_t* d_scales, void* d_workspace, size_t workspace_bytes) {
    if (bad_type(dtype) || n < 0 || n > MAX_ROWS || k < 1 || k > MAX_COLS || o < 1 || o > MAX_COLS || bad_rows(d_x, ld_x, n, k, dtype) || bad_rows(d_w, ld_w, 1, k, dtype) ||
        bad_rows(d_y, ld_y, n, o, dtype) || (d_bias && bad_rows(d_bias, o, 1, o, dtype)) || (d_codes == nullptr) != (d_scales == nullptr) || (d_codes && bad_codes(d_codes)))
        return fail(IBLNERF_ERR_INVALID, "dense_forward: bad arguments (dtype %d, n=%lld, k=%d, o=%d, ld_x=%lld, ld_w=%lld, ld_y=%lld)", dtype, (long long)n, k, o, (long long)ld_x,
                    (long long)ld_w, (long long)ld_y);
    if (too_many_tiles(n, o)) return fail(IBLNERF_ERR_INVALID, "dense_forward: %lld x %d outputs are more than one launch holds", (long long)n, o);
    const size_t need = iblnerf_dense_forward_workspace(dtype, n, k, o);
    if (bad_workspace(d_workspace, workspace_bytes, need))
        return fail(IBLNERF_ERR_INVALID, "dense_forward: a workspace of %zu bytes is needed, %zu given", need, d_workspace ? workspace_bytes : (size_t)0);
    if (n == 0) return IBLNERF_OK;
    DenseRows a{};
    a.a = d_x; a.lda = ld_x; a.w = d_w; a.ldw = ld_w; a.bias = d_bias; a.y = d_y; a.ldy = ld_y; a.codes = d_codes; a.scales = d_scales;
    a.n = n; a.r = k; a.o = o; a.relu = relu != 0; a.is_signed = relu == 0;
    return done("dense_forward", launch_dense_rows(dtype, false, a, d_workspace, (hipStream_t)stream));
}

size_t iblnerf_dense_backward_workspace(int dtype, int64_t n, int k, int o) {
    if (bad_type(dtype) || n < 0 || n > MAX_ROWS || k < 1 || k > MAX_COLS || o < 1 || o > MAX_COLS) return 0;
    const int splits = dense_weight_splits(dtype, n, k, o);
    const size_t weights = splits > 1 ? (size_t)splits * ((size_t)o * k * sizeof(float) + o * sizeof(double)) : 0, input = dense_rows_bytes(dtype, n, o, k);
    return weights > input ? weights : input;      // (one after the other on the stream)
}

int iblnerf_dense_backward(void* stream, int dtype, const void* d_dy, int64_t ld_dy, int64_t n, int k, int o, const uint8_t* d_x_codes, const uint8_t* d_x_scales, int x_is_signed,
                           const uint8_t* d_y_codes, const void* d_w, int64_t ld_w, void* d_dx, int64_t ld_dx, int grad_dtype, void* d_dw, void* d_db, void* d_workspace,
                           size_t workspace_bytes) {
    if (bad_type(dtype) || n < 0 || n > MAX_ROWS || k < 1 || k > MAX_COLS || o < 1 || o > MAX_COLS || bad_rows(d_dy, ld_dy, n, o, dtype) ||
        (d_dx && (bad_rows(d_dx, ld_dx, n, k, dtype) || bad_rows(d_w, ld_w, 1, k, dtype))) || (d_y_codes && bad_codes(d_y_codes)) || (!d_dw && d_db) || (grad_dtype != dtype && grad_dtype != IBLNERF_FLOAT32) ||
        (d_dw && (bad_rows(d_dw, k, 1, k, grad_dtype) || (n > 0 && (bad_codes(d_x_codes) || !d_x_scales)))) || (d_db && bad_rows(d_db, o, 1, o, grad_dtype)))
        return fail(IBLNERF_ERR_INVALID, "dense_backward: bad arguments (dtype %d, n=%lld, k=%d, o=%d, ld_dy=%lld, ld_w=%lld, ld_dx=%lld; weight gradient %s, bias gradient %s)", dtype,
                    (long long)n, k, o, (long long)ld_dy, (long long)ld_w, (long long)ld_dx, d_dw ? "yes" : "no", d_db ? "yes" : "no");
    if (too_many_tiles(n, k) || too_many_tiles(o, k)) return fail(IBLNERF_ERR_INVALID, "dense_backward: %lld x %d inputs are more than one launch holds", (long long)n, k);
    const size_t need = iblnerf_dense_backward_workspace(dtype, n, k, o);
    if (bad_workspace(d_workspace, workspace_bytes, need))
        return fail(IBLNERF_ERR_INVALID, "dense_backward: a workspace of %zu bytes is needed, %zu given", need, d_workspace ? workspace_bytes : (size_t)0);
    DenseRows a{};
    a.a = d_dy; a.lda = ld_dy; a.w = d_w; a.ldw = ld_w; a.open = d_y_codes; a.y = d_dx; a.ldy = ld_dx; a.n = n; a.r = o; a.o = k;
    DenseWeights w{};
    w.dy = d_dy; w.lddy = ld_dy; w.open = d_y_codes; w.x = Checkpoint8{d_x_codes, d_x_scales, x_is_signed != 0}; w.dw = d_dw; w.db = d_db; w.grad32 = grad_dtype == IBLNERF_FLOAT32;
    w.splits = dense_weight_splits(dtype, n, k, o);
    w.bias_part = static_cast<double*>(d_workspace); w.part = reinterpret_cast<float*>(w.bias_part + (size_t)w.splits * o); w.n = n; w.k = k; w.o = o;
    return done("dense_backward", launch_dense_backward(dtype, d_dx ? &a : nullptr, d_dw ? &w : nullptr, d_workspace, (hipStream_t)stream));
}

static bool bad_lookup(int dtype, int64_t v, int d, const void* index, int bits, int64_t n, int64_t per) {
    return bad_type(dtype) || v < 1 || v > MAX_ROWS || d < 1 || d > MAX_COLS || (bits != 32 && bits != 64) || n < 0 || n > MAX_ROWS || per < 1 || per > MAX_ROWS ||
           (n > 0 && n > MAX_ROWS / per) || (n > 0 && (!index || (reinterpret_cast<uintptr_t>(index) & (bits / 8 - 1)) != 0));
}

int iblnerf_lookup(void* stream, int dtype, const void* d_table, int64_t ld_table, int64_t v, int d, const void* d_index, int index_bits, int64_t n, int64_t rows_per_index, float scale,
                   void* d_out, int64_t ld_out) {
    if (bad_lookup(dtype, v, d, d_index, index_bits, n, rows_per_index) || bad_rows(d_table, ld_table, 1, d, dtype) || bad_rows(d_out, ld_out, n, d, dtype))
        return fail(IBLNERF_ERR_INVALID, "lookup: bad arguments (dtype %d, table %lld x %d stride %lld, %lld indices of %d bits, %lld rows each, out stride %lld)", dtype, (long long)v, d,
                    (long long)ld_table, (long long)n, index_bits, (long long)rows_per_index, (long long)ld_out);
    if (n == 0) return IBLNERF_OK;
    return done("lookup", launch_lookup(dtype, Lookup{d_table, ld_table, d_index, index_bits == 64, d_out, ld_out, n, rows_per_index, v, d, scale}, (hipStream_t)stream));
}

size_t iblnerf_lookup_backward_workspace(int64_t n, int64_t rows_per_index, int64_t v, int d) {
    if (n < 0 || n > MAX_ROWS || rows_per_index < 1 || rows_per_index > MAX_ROWS || (n > 0 && n > MAX_ROWS / rows_per_index) || v < 1 || v > MAX_ROWS || d < 1 || d > MAX_COLS) return 0;
    return lookup_backward_bytes(n, rows_per_index, v, d);
}

int iblnerf_lookup_backward(void* stream, int dtype, const void* d_dout, int64_t ld_dout, const void* d_index, int index_bits, int64_t n, int64_t rows_per_index, int64_t v, int d,
                            float scale, void* d_dtable, void* d_workspace, size_t workspace_bytes) {
    if (bad_lookup(dtype, v, d, d_index, index_bits, n, rows_per_index) || bad_rows(d_dout, ld_dout, n, d, dtype) || bad_rows(d_dtable, d, 1, d, dtype))
        return fail(IBLNERF_ERR_INVALID, "lookup_backward: bad arguments (dtype %d, table %lld x %d, %lld indices of %d bits, %lld rows each, stride %lld)", dtype, (long long)v, d,
                    (long long)n, index_bits, (long long)rows_per_index, (long long)ld_dout);
    const size_t need = iblnerf_lookup_backward_workspace(n, rows_per_index, v, d);
    if (bad_workspace(d_workspace, workspace_bytes, n > 0 ? need : 0))
        return fail(IBLNERF_ERR_INVALID, "lookup_backward: a workspace of %zu bytes is needed, %zu given", need, d_workspace ? workspace_bytes : (size_t)0);
    return done("lookup_backward", launch_lookup_backward(dtype, LookupGrad{d_dout, ld_dout, d_index, index_bits == 64, d_dtable, d_workspace, n, rows_per_index, v, d, scale}, (hipStream_t)stream));
}

}  // extern "C"
