// Dense layers of the networks that train layer by layer, and the 8-bit checkpoints their backward pass reads.
//
// CHECKPOINT of an activation [n][k]: per row and block of 32 columns one scale byte s and 32 codes; value = code * 2^(s - 127).  Signed: code in [-127, 127] (two's
// complement), unsigned (what a ReLU leaves): [0, 255].  e = s - 127 is the smallest exponent >= -126 with max|x| <= 127 * 2^e (255 * 2^e), so the codes use 6.98 to
// 7.98 bits of the block's largest entry and an entry is off by at most half a step of 2^e.  A power of two, not max / 255, so that a value has at most 8 significant bits:
// it IS a bfloat16 (and, for an activation that was one, a float16), and the weight gradient's matrix products read it without another rounding.  A positive entry of an
// unsigned checkpoint keeps at least code 1 (off by less than one step instead of half): "code is not zero" is then exactly "the ReLU was open", and no mask is stored.
// A block with a non-finite entry has scale byte 255 and codes 1: all its values are NaN, and its ReLUs count as open.  Rows are padded to 32 columns with zeros.
//
// PRODUCTS.  16-bit types: one v_mfma_f32_32x32x16 per 32 x 32 x 16 block, fp32 accumulation, one rounding to the type at the end.  float32: every operand is cut
// into three bfloat16 parts, each the rest rounded to nearest, x = h + l + r EXACTLY (8 + 8 + 8 bits), and the six products hh + hl + lh + ll + hr + rh are added up in the
// same fp32 accumulator: what is left out (lr + rl + rr) is at most 2^-24 of |x||w|, the size of fp32's own rounding of a product; six 16-bit products take 24 matrix-core
// slots where the fp32 instruction takes 64.  (An infinity in a float32 operand, or a magnitude above bfloat16's largest, 3.39e38, comes out as NaN: its lower parts are
// inf - inf.)  A checkpoint's value is one part by itself: three products.
#include "layer_elems.h"
#include "layers.h"

namespace ibl {

namespace {

// eight elements into the matrix-operand planes in LDS: 16-bit types as they are, float32 as its three bfloat16 parts
template <int T> __device__ __forceinline__ void stage8(unsigned short* dst, int plane, const Raw8<T>& v) {
    if constexpr (T == LT_F32) {
        u32x4 part[3];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float x = as_float(v.q[i >> 1][2 * (i & 1)]), y = as_float(v.q[i >> 1][2 * (i & 1) + 1]);
#pragma unroll
            for (int q = 0; q < 3; ++q) {
                const unsigned h = pack2<LT_BF16>(x, y);
                part[q][i] = h;
                x -= as_float(h << 16);
                y -= as_float(h & 0xffff0000u);
            }
        }
#pragma unroll
        for (int q = 0; q < 3; ++q) *reinterpret_cast<u32x4*>(dst + q * plane) = part[q];
    } else {
        *reinterpret_cast<u32x4*>(dst) = v.q[0];
    }
}

template <int T> __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (T == LT_F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// the product of two operands of PA and PB parts: every pair of parts whose orders add up to less than 3
template <int T, int PA, int PB> __device__ __forceinline__ f32x16 product(const u32x4 (&a)[PA], const u32x4 (&b)[PB], f32x16 c) {
#pragma unroll
    for (int i = PA - 1; i >= 0; --i)
#pragma unroll
        for (int j = PB - 1; j >= 0; --j)
            if (i + j < 3) c = mfma<T>(a[i], b[j], c);
    return c;
}

// Two LDS layouts of an operand tile, 16-bit elements:
// "along": rows of BK reduction elements, the 16-byte chunk c of row i at place c ^ (i / (16 / C) % C), C = BK / 8 — 8 rows x one chunk fall on all banks
template <int BK> __device__ __forceinline__ int along(int i, int c) {
    constexpr int C = BK / 8;
    return i * BK + ((c ^ ((i / (16 / C)) % C)) * 8);
}
// "across": one row of 128 columns for each reduction index; the 64-byte chunk c of row p at place c ^ (p & 3): the transposing read below takes 4 rows x 64 bytes at once
__device__ __forceinline__ int across(int p, int c32) { return p * 128 + ((c32 ^ (p & 3)) * 32); }

// Operand fragments of step ks (16 reduction elements): lane (i = lane & 31, h = lane >> 5) holds elements 8 h .. 8 h + 7 of column / row i of the 32-wide tile
template <int BK> __device__ __forceinline__ u32x4 frag_along(const unsigned short* t, int row0, int ks, int lane) {
    return *reinterpret_cast<const u32x4*>(t + along<BK>(row0 + (lane & 31), 2 * ks + (lane >> 5)));
}
// ds_read_tr16_b64: 16 lanes read 4 rows of 16 columns (8 bytes each) and get column (lane & 15), 4 rows each: two reads make the 8 reduction elements
__device__ __forceinline__ u32x4 frag_across(const unsigned short* t, int c32, int ks, int lane) {
    const int l = lane & 15, half = (lane >> 4) & 1, h = lane >> 5;
    const unsigned short* p = t + across(16 * ks + 8 * h + (l >> 2), c32) + 16 * half + 4 * (l & 3);
    union { s16x4 s[2]; u32x4 u; } v;
    v.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
    v.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * 128));
    return v.u;
}

// Block statistics and codes of 8 of a block's 32 values; the four lanes that hold the block sit side by side (lane & ~3).  Every lane of the four must arrive.
__device__ __forceinline__ void encode8(const float (&f)[8], bool is_signed, u32x2& codes, unsigned& scale) {
    int mag = 0, pos = 0;      // float bits as integers order as the magnitudes do; an infinity or NaN is >= 0x7f800000
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int b = (int)as_bits(f[i]);
        mag = max(mag, b & 0x7fffffff);
        pos = max(pos, b);
    }
    mag = max(mag, __shfl_xor(mag, 1)); mag = max(mag, __shfl_xor(mag, 2));
    pos = max(pos, __shfl_xor(pos, 1)); pos = max(pos, __shfl_xor(pos, 2));
    const int a = is_signed ? mag : pos;
    // 127 = 1.984375 * 2^6 (fraction bits 0x7e0000), 255 = 1.9921875 * 2^7 (0x7f0000)
    const int e = max((a >> 23) - 127 - (is_signed ? 6 : 7) + ((a & 0x7fffff) > (is_signed ? 0x7e0000 : 0x7f0000) ? 1 : 0), -126);
    const bool bad = mag >= 0x7f800000;
    const float inv = as_float(bad ? 0 : (127 - e) << 23);
    unsigned c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int q = (int)rintf(f[i] * inv);
        c[i] = is_signed ? (unsigned)q & 255u : (f[i] > 0.0f ? (unsigned)max(q, 1) : 0u);
    }
#pragma unroll
    for (int g = 0; g < 2; ++g) codes[g] = bad ? 0x01010101u : (c[4 * g] | c[4 * g + 1] << 8 | c[4 * g + 2] << 16 | c[4 * g + 3] << 24);
    scale = bad ? 255u : (unsigned)(e + 127);
}

// the eight values behind codes: (u - off) * step in one exact fused multiply-add (u the code byte, its top bit flipped where signed); scale byte 255 makes step infinite
// and every value NaN
__device__ __forceinline__ void decode8(u32x2 codes, unsigned scale, bool is_signed, float (&f)[8]) {
    const float step = as_float(scale << 23);
    const unsigned flip = is_signed ? 0x80808080u : 0u;
    const float off = (is_signed ? -128.0f : -0.0f) * step;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const unsigned u = ((codes[i >> 2] ^ flip) >> (8 * (i & 3))) & 255u;
        f[i] = __builtin_fmaf((float)u, step, off);
    }
}

// ------------------------------------------------------------------------------------------------------------------------------ Y = act(A B + bias)
// One workgroup = BP rows x BO outputs, 4 waves of (BP / 2) x (BO / 2); D[output][row] so that a lane's accumulators are runs of 4 outputs of ONE row.  The reduction runs
// in steps of BK staged through LDS: the next step's elements travel into registers while this step's products run.
// Neighbouring workgroups of one XCD take the output tiles of the same rows (the rows are read from HBM once and then from that XCD's L2).
template <int T, bool DX, int BP, int BO>
__global__ __launch_bounds__(256, 2) void k_dense_rows(DenseRows a) {
    constexpr int PARTS = T == LT_F32 ? 3 : 1, BK = T == LT_F32 ? 32 : 64;
    constexpr int TP = BP / 64, TO = BO / 64;                      // 32-wide tiles of a wave
    constexpr int XC = BP * BK / 8 / 256, WC = BO * BK / 8 / 256;  // 8-element chunks a thread stages
    constexpr int XPLANE = BP * BK, WPLANE = BO * BK;
    constexpr int RS = (BO / 2) * Bytes<T>::v + 16;                // epilogue: bytes of a row in a wave's LDS window of 32 rows
    constexpr int STAGE = PARTS * (XPLANE + WPLANE) * 2, OUT = 4 * 32 * RS;
    static_assert(!DX || BO == 128, "the across layout has rows of 128 columns");
    __shared__ __attribute__((aligned(16))) char lds[STAGE > OUT ? STAGE : OUT];
    __shared__ float bias[BO];
    unsigned short* xt = reinterpret_cast<unsigned short*>(lds);
    unsigned short* wt = xt + PARTS * XPLANE;

    const int ot = (a.o + BO - 1) / BO;
    const long j = blockIdx.x >> 3;
    const long pt = (j / ot) * 8 + (blockIdx.x & 7);
    const long p0 = pt * BP;
    const int o0 = (int)(j % ot) * BO;
    if (p0 >= a.n) return;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int wp = (wave >> 1) * (BP / 2), wo = (wave & 1) * (BO / 2);
    if (t < BO) {
        float b = 0.0f;
        if (!DX && a.bias && o0 + t < a.o) {
            if constexpr (T == LT_F32) b = static_cast<const float*>(a.bias)[o0 + t];
            else if constexpr (T == LT_BF16) b = as_float((unsigned)static_cast<const unsigned short*>(a.bias)[o0 + t] << 16);
            else b = (float)static_cast<const _Float16*>(a.bias)[o0 + t];
        }
        bias[t] = b;
    }

    const int r32 = (a.r + 31) & ~31;
    Raw8<T> xr[XC], wr[WC];
    u32x2 cr[XC];
    auto load = [&](int k0) {
#pragma unroll
        for (int i = 0; i < XC; ++i) {
            const int c = t + 256 * i, row = c / (BK / 8), k = k0 + 8 * (c % (BK / 8));
            const long p = p0 + row;
            const bool in = p < a.n;
            xr[i] = in ? load8<T>(static_cast<const char*>(a.a) + p * a.lda * Bytes<T>::v, k, a.r) : zero8<T>();
            if (DX) {
                cr[i] = u32x2{0x01010101u, 0x01010101u};
                if (a.open && in && k < r32) cr[i] = *reinterpret_cast<const u32x2*>(a.open + p * r32 + k);
            }
        }
#pragma unroll
        for (int i = 0; i < WC; ++i) {
            const int c = t + 256 * i;
            if (!DX) {
                const int row = c / (BK / 8), k = k0 + 8 * (c % (BK / 8));
                wr[i] = o0 + row < a.o ? load8<T>(static_cast<const char*>(a.w) + (o0 + row) * a.ldw * Bytes<T>::v, k, a.r) : zero8<T>();
            } else {
                const int row = c / (BO / 8), col = o0 + 8 * (c % (BO / 8));
                wr[i] = k0 + row < a.r ? load8<T>(static_cast<const char*>(a.w) + (k0 + row) * a.ldw * Bytes<T>::v, col, a.o) : zero8<T>();
            }
        }
    };
    auto stage = [&]() {
#pragma unroll
        for (int i = 0; i < XC; ++i) {
            const int c = t + 256 * i;
            if (DX) close8<T>(xr[i], cr[i]);
            stage8<T>(xt + along<BK>(c / (BK / 8), c % (BK / 8)), XPLANE, xr[i]);
        }
#pragma unroll
        for (int i = 0; i < WC; ++i) {
            const int c = t + 256 * i;
            if (!DX) stage8<T>(wt + along<BK>(c / (BK / 8), c % (BK / 8)), WPLANE, wr[i]);
            else stage8<T>(wt + across(c / (BO / 8), (c % (BO / 8)) >> 2) + 8 * (c & 3), WPLANE, wr[i]);
        }
    };

    f32x16 acc[TO][TP];
#pragma unroll
    for (int i = 0; i < TO; ++i)
#pragma unroll
        for (int k = 0; k < TP; ++k) acc[i][k] = f32x16{0};
    load(0);
    for (int k0 = 0; k0 < a.r; k0 += BK) {
        if (k0) __syncthreads();
        stage();
        __syncthreads();
        if (k0 + BK < a.r) load(k0 + BK);
#pragma unroll
        for (int ks = 0; ks < BK / 16; ++ks) {
            u32x4 x[TP][PARTS];
#pragma unroll
            for (int i = 0; i < TP; ++i)
#pragma unroll
                for (int q = 0; q < PARTS; ++q) x[i][q] = frag_along<BK>(xt + q * XPLANE, wp + 32 * i, ks, lane);
#pragma unroll
            for (int i = 0; i < TO; ++i) {
                u32x4 w[PARTS];
#pragma unroll
                for (int q = 0; q < PARTS; ++q)
                    w[q] = DX ? frag_across(wt + q * WPLANE, (wo >> 5) + i, ks, lane) : frag_along<BK>(wt + q * WPLANE, wo + 32 * i, ks, lane);
#pragma unroll
                for (int k = 0; k < TP; ++k) acc[i][k] = product<T, PARTS, PARTS>(w, x[k], acc[i][k]);
            }
        }
    }
    __syncthreads();

    // 32 rows at a time through the wave's own window of LDS: rounded outputs in, whole row pieces out (16 bytes a lane) with their checkpoint
    char* win = lds + wave * 32 * RS;
    const int h = lane >> 5;
#pragma unroll
    for (int k = 0; k < TP; ++k) {
#pragma unroll
        for (int i = 0; i < TO; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[e] = acc[i][k][4 * g + e] + bias[wo + 32 * i + 8 * g + 4 * h + e];
                    if (!DX && a.relu) v[e] = v[e] < 0.0f ? 0.0f : v[e];      // (a NaN stays)
                }
                char* dst = win + (lane & 31) * RS + (32 * i + 8 * g + 4 * h) * Bytes<T>::v;
                if constexpr (T == LT_F32) {
                    *reinterpret_cast<u32x4*>(dst) = u32x4{as_bits(v[0]), as_bits(v[1]), as_bits(v[2]), as_bits(v[3])};
                } else {
                    *reinterpret_cast<u32x2*>(dst) = u32x2{pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])};
                }
            }
        __builtin_amdgcn_wave_barrier();
        constexpr int LPR = BO / 16;                       // lanes a row (8 outputs each)
#pragma unroll
        for (int pass = 0; pass < 32 * LPR / 64; ++pass) {
            const int row = pass * (64 / LPR) + lane / LPR, c = 8 * (lane % LPR);
            const long p = p0 + wp + 32 * k + row;
            const int o = o0 + wo + c;
            Raw8<T> v;
            v.q[0] = *reinterpret_cast<const u32x4*>(win + row * RS + c * Bytes<T>::v);
            if constexpr (T == LT_F32) v.q[1] = *reinterpret_cast<const u32x4*>(win + row * RS + c * 4 + 16);
            const bool in = p < a.n && o < a.o;
            if (in) store8<T>(static_cast<char*>(a.y) + p * a.ldy * Bytes<T>::v, o, a.o, v);
            if (!DX && a.codes) {
                float f[8];
                to_floats<T>(v, f);
#pragma unroll
                for (int e = 0; e < 8; ++e) if (o + e >= a.o) f[e] = 0.0f;
                u32x2 codes; unsigned scale;
                encode8(f, a.is_signed != 0, codes, scale);
                const int o32 = (a.o + 31) & ~31;
                if (p < a.n && o < o32) {
                    *reinterpret_cast<u32x2*>(a.codes + p * o32 + o) = codes;
                    if ((c & 31) == 0) a.scales[p * (o32 >> 5) + (o >> 5)] = (uint8_t)scale;
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// --------------------------------------------------------------------------------------------------------------------------------- dW = dZ^T X, db
// One workgroup = 128 outputs x 128 input columns over its piece of the rows, 4 waves of 64 x 64; BR rows a step.  Both operands lie with the REDUCTION index as the row, as
// they do in memory, and are turned by the transposing LDS read.  The pieces' sums go to `part` and are added in order by k_dense_weights_sum: no atomics, the same
// bits every time.
template <int T>
__global__ __launch_bounds__(256, 2) void k_dense_weights(DenseWeights a) {
    constexpr int PARTS = T == LT_F32 ? 3 : 1, BR = T == LT_F32 ? 32 : 64;
    constexpr int PLANE = BR * 128, NC = BR * 16 / 256;
    __shared__ __attribute__((aligned(16))) unsigned short lds[(PARTS + 1) * PLANE];
    unsigned short* zt = lds;
    unsigned short* xt = lds + PARTS * PLANE;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int kt = (a.k + 127) / 128, ot = (a.o + 127) / 128, tiles = kt * ot;
    const long j = blockIdx.x >> 3;
    const int split = (int)(j / tiles) * 8 + (blockIdx.x & 7);
    if (split >= a.splits) return;
    const int tile = (int)(j % tiles), k0 = (tile % kt) * 128, o0 = (tile / kt) * 128;
    const long steps = (a.n + BR - 1) / BR;
    const long s0 = steps * split / a.splits, s1 = steps * (split + 1) / a.splits;
    const int k32 = (a.k + 31) & ~31, o32 = (a.o + 31) & ~31;
    const int cc = 8 * (t & 15);                       // the thread's 8 columns of either tile (the same in every step), rows t / 16 + 16 i
    const bool sums = a.db != nullptr && k0 == 0;

    Raw8<T> zr[NC];
    u32x2 cr[NC], xc[NC];
    unsigned xs[NC];
    auto load = [&](long step) {
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const long p = step * BR + (t >> 4) + 16 * i;
            const bool in = p < a.n;
            zr[i] = in ? load8<T>(static_cast<const char*>(a.dy) + p * a.lddy * Bytes<T>::v, o0 + cc, a.o) : zero8<T>();
            cr[i] = u32x2{0x01010101u, 0x01010101u};
            if (a.open && in && o0 + cc < o32) cr[i] = *reinterpret_cast<const u32x2*>(a.open + p * o32 + o0 + cc);
            const bool inx = in && k0 + cc < k32;
            xc[i] = inx ? *reinterpret_cast<const u32x2*>(a.x.codes + p * k32 + k0 + cc) : u32x2{0, 0};
            xs[i] = inx ? a.x.scales[p * (k32 >> 5) + ((k0 + cc) >> 5)] : 256u;      // (256: beyond the rows or columns)
        }
    };
    // the bias gradient is one sum over all rows, with nothing to average an error out: 64 bits from one step to the next (and within a step for float32, whose terms fill fp32)
    double bs[8] = {0., 0., 0., 0., 0., 0., 0., 0.};
    auto stage = [&]() {
        float few[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int at = across((t >> 4) + 16 * i, (t & 15) >> 2) + 8 * (t & 3);
            close8<T>(zr[i], cr[i]);
            stage8<T>(zt + at, PLANE, zr[i]);
            if (sums) {
                float f[8];
                to_floats<T>(zr[i], f);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if constexpr (T == LT_F32) bs[e] += (double)f[e];
                    else few[e] += f[e];
                }
            }
            float f[8];
            decode8(xc[i], xs[i] & 255u, a.x.is_signed != 0, f);
            u32x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e)      // a value has at most 8 significant bits: its upper 16 bits are all of it
                v[e] = T == LT_F16 ? pack2<LT_F16>(f[2 * e], f[2 * e + 1])
                                   : __builtin_amdgcn_perm(as_bits(f[2 * e + 1]), as_bits(f[2 * e]), 0x07060302u);
            if (xs[i] == 256u) v = u32x4{0, 0, 0, 0};
            *reinterpret_cast<u32x4*>(xt + at) = v;
        }
        if (T != LT_F32 && sums)
#pragma unroll
            for (int e = 0; e < 8; ++e) bs[e] += (double)few[e];
    };

    const int wo = (wave >> 1) * 2, wk = (wave & 1) * 2;      // the wave's first 32-wide tile of either side
    f32x16 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) acc[i][k] = f32x16{0};
    if (s0 < s1) load(s0);
    for (long s = s0; s < s1; ++s) {
        if (s > s0) __syncthreads();
        stage();
        __syncthreads();
        if (s + 1 < s1) load(s + 1);
#pragma unroll
        for (int ks = 0; ks < BR / 16; ++ks) {
            u32x4 x[2][1];
#pragma unroll
            for (int k = 0; k < 2; ++k) x[k][0] = frag_across(xt, wk + k, ks, lane);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                u32x4 z[PARTS];
#pragma unroll
                for (int q = 0; q < PARTS; ++q) z[q] = frag_across(zt + q * PLANE, wo + i, ks, lane);
#pragma unroll
                for (int k = 0; k < 2; ++k) acc[i][k] = product<T, PARTS, 1>(z, x[k], acc[i][k]);
            }
        }
    }
    const bool last = a.splits == 1;
    auto put = [&](void* to, long at, float v) {
        if (T == LT_F32 || a.grad32) static_cast<float*>(to)[at] = v;
        else static_cast<unsigned short*>(to)[at] = (unsigned short)pack2<T == LT_F32 ? LT_F16 : T>(v, 0.0f);
    };
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int o = o0 + 32 * (wo + i) + (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5), c = k0 + 32 * (wk + k) + (lane & 31);
                if (o < a.o && c < a.k) {
                    if (last) put(a.dw, (long)o * a.k + c, acc[i][k][r]);
                    else a.part[((long)split * a.o + o) * a.k + c] = acc[i][k][r];
                }
            }
    if (sums) {      // 16 threads hold sums of the same 8 columns
        __syncthreads();
        double* f = reinterpret_cast<double*>(lds);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[(t >> 4) * 128 + cc + e] = bs[e];
        __syncthreads();
        if (t < 128 && o0 + t < a.o) {
            double s = 0.0;
#pragma unroll
            for (int i = 0; i < 16; ++i) s += f[i * 128 + t];
            if (last) put(a.db, o0 + t, (float)s);
            else a.bias_part[(long)split * a.o + o0 + t] = s;
        }
    }
}

template <int T> __global__ __launch_bounds__(256) void k_dense_weights_sum(DenseWeights a) {
    const long nw = (long)a.o * a.k, i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= nw + (a.db ? a.o : 0)) return;
    const bool bias = i >= nw;
    const long at = bias ? i - nw : i;
    double s = 0.0;
    if (bias) {
        for (int q = 0; q < a.splits; ++q) s += a.bias_part[(long)q * a.o + at];
    } else {
#pragma unroll 8
        for (int q = 0; q < a.splits; ++q) s += (double)a.part[q * nw + at];
    }
    void* to = bias ? a.db : a.dw;
    if (T == LT_F32 || a.grad32) static_cast<float*>(to)[at] = (float)s;
    else static_cast<unsigned short*>(to)[at] = (unsigned short)pack2<T == LT_F32 ? LT_F16 : T>((float)s, 0.0f);
}

// ------------------------------------------------------------------------------------------------------------------------- checkpoints on their own
template <int T> __global__ __launch_bounds__(256) void k_checkpoint(const char* x, long ld, long n, int k, int is_signed, uint8_t* codes, uint8_t* scales) {
    const int cpr = ((k + 31) >> 5) * 4;      // 8-column chunks a row; a block's four lie in four neighbouring lanes
    const long total = n * cpr;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < ((total + 63) & ~63L); i += (long)gridDim.x * 256) {      // whole waves: encode8 exchanges between lanes
        const bool in = i < total;
        const long p = in ? i / cpr : 0;
        const int c = 8 * (int)(in ? i - p * cpr : 0);
        float f[8];
        to_floats<T>(in ? load8<T>(x + p * ld * Bytes<T>::v, c, k) : zero8<T>(), f);
        u32x2 q; unsigned s;
        encode8(f, is_signed != 0, q, s);
        if (in) {
            *reinterpret_cast<u32x2*>(codes + 8 * i) = q;
            if ((c & 31) == 0) scales[i >> 2] = (uint8_t)s;
        }
    }
}

template <int T> __global__ __launch_bounds__(256) void k_checkpoint_values(Checkpoint8 a, long n, int k, char* out, long ld) {
    const int cpr = ((k + 31) >> 5) * 4;
    const long total = n * cpr;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
        const long p = i / cpr;
        const int c = 8 * (int)(i - p * cpr);
        if (c >= k) continue;
        float f[8];
        decode8(*reinterpret_cast<const u32x2*>(a.codes + 8 * i), a.scales[i >> 2], a.is_signed != 0, f);
        store8<T>(out + p * ld * Bytes<T>::v, c, k, from_floats<T>(f));
    }
}

template <int T> hipError_t dense_rows(bool dx, const DenseRows& a, hipStream_t s) {
    const long pt = (a.n + 127) / 128, ot = (a.o + 127) / 128;
    const dim3 grid((unsigned)((pt + 7) / 8 * 8 * ot));
    if (dx) hipLaunchKernelGGL((k_dense_rows<T, true, 128, 128>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_dense_rows<T, false, 128, 128>), grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

template <int T> hipError_t dense_weights(const DenseWeights& a, hipStream_t s) {
    const long tiles = (long)((a.k + 127) / 128) * ((a.o + 127) / 128);
    hipLaunchKernelGGL((k_dense_weights<T>), dim3((unsigned)((a.splits + 7) / 8 * 8 * tiles)), dim3(256), 0, s, a);
    if (a.splits > 1) {
        const long m = (long)a.o * a.k + a.o;
        hipLaunchKernelGGL((k_dense_weights_sum<T>), dim3((unsigned)((m + 255) / 256)), dim3(256), 0, s, a);
    }
    return hipGetLastError();
}

unsigned chunk_grid(long n, int k) {
    const long blocks = (n * (((k + 31) >> 5) * 4) + 255) / 256;
    return (unsigned)(blocks < 16384 ? blocks : 16384);
}

}  // namespace

int dense_weight_splits(long n, int k, int o, int type) {
    const long tiles = (long)((k + 127) / 128) * ((o + 127) / 128), steps = (n + (type == LT_F32 ? 31 : 63)) / (type == LT_F32 ? 32 : 64);
    long s = 1024 / tiles;      // four workgroups for each of the 256 compute units
    if (s > steps) s = steps;
    return (int)(s < 1 ? 1 : s);
}

hipError_t launch_dense_rows(int type, bool input_gradient, const DenseRows& a, hipStream_t s) {
    return type == LT_F32 ? dense_rows<LT_F32>(input_gradient, a, s) : type == LT_BF16 ? dense_rows<LT_BF16>(input_gradient, a, s) : dense_rows<LT_F16>(input_gradient, a, s);
}

hipError_t launch_dense_weights(int type, const DenseWeights& a, hipStream_t s) {
    return type == LT_F32 ? dense_weights<LT_F32>(a, s) : type == LT_BF16 ? dense_weights<LT_BF16>(a, s) : dense_weights<LT_F16>(a, s);
}

hipError_t launch_checkpoint(int type, const void* x, long ld, long n, int k, int is_signed, uint8_t* codes, uint8_t* scales, hipStream_t s) {
    const dim3 g(chunk_grid(n, k)), b(256);
    const char* p = static_cast<const char*>(x);
    if (type == LT_F32) hipLaunchKernelGGL((k_checkpoint<LT_F32>), g, b, 0, s, p, ld, n, k, is_signed, codes, scales);
    else if (type == LT_BF16) hipLaunchKernelGGL((k_checkpoint<LT_BF16>), g, b, 0, s, p, ld, n, k, is_signed, codes, scales);
    else hipLaunchKernelGGL((k_checkpoint<LT_F16>), g, b, 0, s, p, ld, n, k, is_signed, codes, scales);
    return hipGetLastError();
}

hipError_t launch_checkpoint_values(int type, const Checkpoint8& c, long n, int k, void* out, long ld, hipStream_t s) {
    const dim3 g(chunk_grid(n, k)), b(256);
    char* p = static_cast<char*>(out);
    if (type == LT_F32) hipLaunchKernelGGL((k_checkpoint_values<LT_F32>), g, b, 0, s, c, n, k, p, ld);
    else if (type == LT_BF16) hipLaunchKernelGGL((k_checkpoint_values<LT_BF16>), g, b, 0, s, c, n, k, p, ld);
    else hipLaunchKernelGGL((k_checkpoint_values<LT_F16>), g, b, 0, s, c, n, k, p, ld);
    return hipGetLastError();
}

}  // namespace ibl
