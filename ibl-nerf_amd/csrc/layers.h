// Argument blocks and launchers of the trainable-layer operators (dense_kernel.hip, lookup_kernel.hip), called by layers_api.cpp (include/iblnerf_layers.h).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace ibl {

enum LayerType { LT_F32 = 0, LT_BF16 = 1, LT_F16 = 2 };

// an 8-bit checkpoint [n][k]: codes [n][32 kb], scale bytes [n][kb], kb = ceil(k / 32) (the format: dense_kernel.hip)
struct Checkpoint8 {
    const uint8_t* codes;
    const uint8_t* scales;
    int is_signed;
};

// Y [n][o] = act(A [n][r] B + bias), A row-major; B = W [o][r] (forward) or W [r][o] (the input gradient: A = dY where `open` is nonzero)
struct DenseRows {
    const void* a; long lda;
    const void* w; long ldw;
    const void* bias;            // [o] or null (forward)
    const uint8_t* open;         // [n][32 ceil(r / 32)] codes of the layer's output, or null (input gradient)
    void* y; long ldy;
    uint8_t* codes; uint8_t* scales;      // the checkpoint of y, or null (forward)
    long n; int r, o;
    int relu, is_signed;
};
size_t dense_rows_bytes(int type, long n, int r, int o);      // scratch memory of the launch
hipError_t launch_dense_rows(int type, bool input_gradient, const DenseRows& a, void* ws, hipStream_t s);

// dW [o][k] = sum_p dZ[p][o] X[p][k], db [o] = sum_p dZ[p][o];  dZ = dY where `open` is nonzero (or everywhere: null)
struct DenseWeights {
    const void* dy; long lddy;
    const uint8_t* open;
    Checkpoint8 x;
    void* dw; void* db;          // [o][k], [o] contiguous (db may be null), of the activations' type, or float32 (grad32)
    int grad32;
    double* bias_part;           // [splits][o]
    float* part;                 // [splits][o][k] (neither is read or written with one split)
    long n; int k, o;
    int splits;
};
int dense_weight_splits(int type, long n, int k, int o);      // how many pieces the rows are cut into (a function of the sizes alone: results repeat bit for bit)
// both gradients of a layer, or one (null: not asked for); ws is the input gradient's scratch memory
hipError_t launch_dense_backward(int type, const DenseRows* x, const DenseWeights* w, void* ws, hipStream_t s);

hipError_t launch_checkpoint(int type, const void* x, long ld, long n, int k, int is_signed, uint8_t* codes, uint8_t* scales, hipStream_t s);
hipError_t launch_checkpoint_values(int type, const Checkpoint8& c, long n, int k, void* out, long ld, hipStream_t s);

// out [n * per][d] = scale * table[index[row / per]]
struct Lookup {
    const void* table; long ld_table;
    const void* index; int index64;
    void* out; long ld_out;
    long n; long per; long v; int d;
    float scale;
};
hipError_t launch_lookup(int type, const Lookup& a, hipStream_t s);

// dtable [v][d] = scale * sum of dout over each token's rows
struct LookupGrad {
    const void* dout; long ld_dout;
    const void* index; int index64;
    void* dtable;
    void* ws;
    long n; long per; long v; int d;
    float scale;
};
size_t lookup_backward_bytes(long n, long per, long v, int d);
hipError_t launch_lookup_backward(int type, const LookupGrad& a, hipStream_t s);

}  // namespace ibl
