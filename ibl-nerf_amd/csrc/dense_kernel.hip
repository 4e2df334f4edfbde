// Dense layers of the networks that train layer by layer, and the 8-bit checkpoints their backward pass reads.
//
// CHECKPOINT of an activation [n][k]: per row and block of 32 columns one scale byte s and 32 codes; value = code * 2^(s - 127).  Signed: code in [-127, 127] (two's
// complement), unsigned (what a ReLU leaves): [0, 255].  e = s - 127 is the smallest exponent >= -126 with max|x| <= 127 * 2^e (255 * 2^e), so the codes use 6.98 to
// 7.98 bits of the block's largest entry and an entry is off by at most half a step of 2^e.  A power of two, not max / 255, so that a value has at most 8 significant bits:
// it IS a bfloat16 (and, for an activation that was one, a float16: but for the upper ends of their ranges, see decode8_large), and the weight gradient's matrix products read it without
// another rounding.  A positive entry of an
// unsigned checkpoint keeps at least code 1 (off by less than one step instead of half): "code is not zero" is then exactly "the ReLU was open", and no mask is stored.
// A block with a non-finite entry has scale byte 255 and codes 1: all its values are NaN, and its ReLUs count as open.  Rows are padded to 32 columns with zeros.
//
// PRODUCTS.  16-bit types: one v_mfma_f32_32x32x16 per 32 x 32 x 16 block, fp32 accumulation, one rounding to the type at the end.  float32: every operand is cut
// into three bfloat16 parts, each the rest rounded to nearest, x = h + l + r EXACTLY (8 + 8 + 8 bits; below 2^-110 the last part is a multiple of 2^-133: off by up to 2^-134), and the six products hh + hl + lh + ll + hr + rh are added up in the
// same fp32 accumulator: what is left out (lr + rl + rr) is at most 2^-24 of |x||w|, the size of fp32's own rounding of a product; six 16-bit products take 24 matrix-core
// slots where the fp32 instruction takes 64.  (An infinity in a float32 operand, or a magnitude above bfloat16's largest, 3.39e38, comes out as NaN: its lower parts are
// inf - inf.)  A checkpoint's value is one part by itself: three products.
#include <atomic>

#include "layer_elems.h"
#include "layers.h"

#include <type_traits>

namespace ibl {

namespace {

// eight elements as matrix operands: 16-bit types as they are, float32 as its three bfloat16 parts
template <int T> struct Parts { static constexpr int n = T == LT_F32 ? 3 : 1; };
template <int T> __device__ __forceinline__ void parts_of(const Raw8<T>& v, u32x4 (&part)[Parts<T>::n]) {
    if constexpr (T == LT_F32) {
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
    } else {
        part[0] = v.q[0];
    }
}
// ... into their planes in LDS
template <int T> __device__ __forceinline__ void stage8(unsigned short* dst, int plane, const Raw8<T>& v) {
    u32x4 part[Parts<T>::n];
    parts_of<T>(v, part);
#pragma unroll
    for (int q = 0; q < Parts<T>::n; ++q) *reinterpret_cast<u32x4*>(dst + q * plane) = part[q];
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
// "across": one row of W columns for each reduction index; the 64-byte chunk c of row p at place c ^ (p & 3): the transposing read below takes 4 rows x 64 bytes at once
// (rows of one chunk lie side by side as they are)
template <int W> __device__ __forceinline__ int across(int p, int c32) { return p * W + ((c32 ^ (p & 3 & (W / 32 - 1))) * 32); }

// Operand fragments of step ks (16 reduction elements): lane (i = lane & 31, h = lane >> 5) holds elements 8 h .. 8 h + 7 of column / row i of the 32-wide tile
template <int BK> __device__ __forceinline__ u32x4 frag_along(const unsigned short* t, int row0, int ks, int lane) {
    return *reinterpret_cast<const u32x4*>(t + along<BK>(row0 + (lane & 31), 2 * ks + (lane >> 5)));
}
// ds_read_tr16_b64: 16 lanes read 4 rows of 16 columns (8 bytes each) and get column (lane & 15), 4 rows each: two reads make the 8 reduction elements
template <int W> __device__ __forceinline__ u32x4 frag_across(const unsigned short* t, int c32, int ks, int lane) {
    const int l = lane & 15, half = (lane >> 4) & 1, h = lane >> 5;
    const unsigned short* p = t + across<W>(16 * ks + 8 * h + (l >> 2), c32) + 16 * half + 4 * (l & 3);
    union { s16x4 s[2]; u32x4 u; } v;
    v.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
    v.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * W));
    return v.u;
}

// the largest of the four lanes side by side (lane & ~3), in each of them
__device__ __forceinline__ unsigned max_of_4(unsigned x) {
    x = max(x, (unsigned)__builtin_amdgcn_mov_dpp((int)x, 0xb1, 0xf, 0xf, true));      // lanes 1 0 3 2
    return max(x, (unsigned)__builtin_amdgcn_mov_dpp((int)x, 0x4e, 0xf, 0xf, true));   // lanes 2 3 0 1
}

// A block's largest magnitude and the value that sets its step (the largest positive one of an unsigned checkpoint), as bits of its type.  Magnitudes are compared as integers:
// a value's bits without the sign order as the values do, and an infinity or NaN is at least the infinity's.
struct Block { unsigned mag, top; };
template <int T, int N> __device__ __forceinline__ Block block_of(const Raw8<T> (&v)[N], bool is_signed) {
    Block b;
    if constexpr (T == LT_F32) {
        unsigned mag = 0;
        int pos = 0;
#pragma unroll
        for (int i = 0; i < 8 * N; ++i) {
            const unsigned u = v[i >> 3].q[(i & 7) >> 2][i & 3];
            mag = max(mag, u & 0x7fffffffu);
            pos = max(pos, (int)u);
        }
        b = Block{mag, is_signed ? mag : (unsigned)pos};
    } else {
        u16x2 m = {0, 0};
        s16x2 p = {0, 0};
#pragma unroll
        for (int i = 0; i < 4 * N; ++i) {
            const unsigned u = v[i >> 2].q[0][i & 3], c = u & 0x7fff7fffu;
            m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, c));
            p = __builtin_elementwise_max(p, __builtin_bit_cast(s16x2, u));
        }
        b.mag = max((unsigned)m[0], (unsigned)m[1]);
        b.top = is_signed ? b.mag : (unsigned)max((int)p[0], (int)p[1]);
    }
    return b;
}

struct Step { float inv; unsigned scale; bool bad; };
template <int T> __device__ __forceinline__ Step step_of(const Block& b, bool is_signed) {
    const bool bad = b.mag >= (T == LT_F32 ? 0x7f800000u : T == LT_BF16 ? 0x7f80u : 0x7c00u);
    const unsigned top = T == LT_F32 ? b.top : T == LT_BF16 ? b.top << 16 : as_bits(half_float(b.top));
    // 127 = 1.984375 * 2^6 (fraction bits 0x7e0000), 255 = 1.9921875 * 2^7 (0x7f0000)
    const int e = max((int)(top >> 23) - 127 - (is_signed ? 6 : 7) + ((top & 0x7fffffu) > (is_signed ? 0x7e0000u : 0x7f0000u) ? 1 : 0), -126);
    return Step{as_float(bad ? 0u : (unsigned)(127 - e) << 23), bad ? 255u : (unsigned)(e + 127), bad};
}

template <int T> __device__ __forceinline__ u32x2 codes_of(const Raw8<T>& v, const Step& s, bool is_signed) {
    float f[8];
    to_floats<T>(v, f);
    u32x2 codes;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        unsigned c = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float u = f[4 * g + i] * s.inv;
            if (is_signed) u = rintf(u) + 128.0f;                                              // (the top bit flipped back below)
            else u = fmaxf(u, __builtin_amdgcn_fmed3f(ceilf(f[4 * g + i]), 0.0f, 1.0f));       // a positive value, however small, keeps at least code 1
            c = __builtin_amdgcn_cvt_pk_u8_f32(u, i, c);                                       // rounds to nearest, ties to even; below zero: 0
        }
        codes[g] = s.bad ? 0x01010101u : is_signed ? c ^ 0x80808080u : c;
    }
    return codes;
}

// Codes and scale byte of 8 of a block's 32 values; the four lanes that hold the block sit side by side, and all of them must arrive
template <int T> __device__ __forceinline__ void encode8(const Raw8<T>& v, bool is_signed, u32x2& codes, unsigned& scale) {
    const Raw8<T> one[1] = {v};
    Block b = block_of<T, 1>(one, is_signed);
    b.mag = max_of_4(b.mag);
    b.top = max_of_4(b.top);
    const Step s = step_of<T>(b, is_signed);
    codes = codes_of<T>(v, s, is_signed);
    scale = s.scale;
}

// the eight values behind codes: (u - off) * step in one exact fused multiply-add (u the code byte, its top bit flipped where signed); scale byte 255 makes step infinite and every
// value NaN.  Not for the blocks of large_block
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
// The upper end of T's range.  An entry may be coded as one step beyond it: 2^128 (float32, bfloat16: read as 255 * 2^120, bfloat16's largest) or 65536 (float16: read as
// 65504), so that a finite activation stays finite; and from step 2^121 on decode8's offset, 128 * step, is beyond float32: here the difference comes first.  Blocks whose values
// stay below 2^16 or 2^128 are none of these.
template <int T> __device__ __forceinline__ bool large_block(unsigned scale) {
    constexpr unsigned FIRST = T == LT_F16 ? 127 + 9 : 127 + 121;      // 128 steps of 2^9 are 65536, of 2^121 are 2^128
    return scale - FIRST < 255 - FIRST;
}
template <int T> __device__ __forceinline__ void decode8_large(u32x2 codes, unsigned scale, bool is_signed, float (&f)[8]) {
    asm volatile("" : "+v"(codes));      // (shared with decode8, the converted codes stay in registers across the branch: the widest weight tiles spill)
    const float step = as_float(scale << 23), most = T == LT_F16 ? 65504.0f : 0x1.fep+127f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const unsigned u = (codes[i >> 2] >> (8 * (i & 3))) & 255u;
        const float v = (float)(is_signed ? (int)(signed char)u : (int)u) * step;
        f[i] = T == LT_F16 && __builtin_fabsf(v) != 65536.0f ? v : __builtin_amdgcn_fmed3f(v, -most, most);
    }
}

// The end of a Y tile: a wave's TP x 32 rows, TO x 32 outputs from o0 on.  32 rows at a time through the wave's own window of LDS: rounded outputs in, whole row pieces out
// (16 bytes a lane) with their checkpoint.
template <int TO, int T> struct Window { static constexpr int row = 32 * TO * Bytes<T>::v + 16, bytes = 32 * row; };
template <int T, bool DX, int TO, int TP>
__device__ __forceinline__ void write_rows(const DenseRows& a, const f32x16 (&acc)[TO][TP], char* win, long p0, int o0, int lane) {
    constexpr int RS = Window<TO, T>::row, LPR = 4 * TO;      // lanes a row (8 outputs each)
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
                    v[e] = acc[i][k][4 * g + e];
                    if (!DX && a.relu) v[e] = __builtin_elementwise_maximum(v[e], 0.0f);      // (a NaN stays, -0 becomes 0)
                }
                char* dst = win + (lane & 31) * RS + (32 * i + 8 * g + 4 * h) * Bytes<T>::v;
                if constexpr (T == LT_F32) *reinterpret_cast<u32x4*>(dst) = u32x4{as_bits(v[0]), as_bits(v[1]), as_bits(v[2]), as_bits(v[3])};
                else *reinterpret_cast<u32x2*>(dst) = u32x2{pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])};
            }
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int pass = 0; pass < 32 * LPR / 64; ++pass) {      // (unrolled it takes registers that the products' loop then spills)
            const int at = pass * 64 + lane, row = at / LPR, c = 8 * (at % LPR);
            const long p = p0 + 32 * k + row;
            const int o = o0 + c;
            Raw8<T> v;
            v.q[0] = *reinterpret_cast<const u32x4*>(win + row * RS + c * Bytes<T>::v);
            if constexpr (T == LT_F32) v.q[1] = *reinterpret_cast<const u32x4*>(win + row * RS + c * 4 + 16);
            if (p < a.n && o < a.o) store8<T>(static_cast<char*>(a.y) + p * a.ldy * Bytes<T>::v, o, a.o, v);
            if (!DX && a.codes) {
                if (o + 8 > a.o) {      // (columns beyond the layer's outputs are coded 0)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (o + e >= a.o) {
                            if constexpr (T == LT_F32) v.q[e >> 2][e & 3] = 0;
                            else v.q[0][e >> 1] &= (e & 1) ? 0x0000ffffu : 0xffff0000u;
                        }
                }
                u32x2 codes; unsigned scale;
                encode8<T>(v, a.is_signed != 0, codes, scale);
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

template <int T> __device__ __forceinline__ float bias_at(const DenseRows& a, int o) {
    if (!a.bias || o >= a.o) return 0.0f;
    if constexpr (T == LT_F32) return static_cast<const float*>(a.bias)[o];
    else if constexpr (T == LT_BF16) return as_float((unsigned)static_cast<const unsigned short*>(a.bias)[o] << 16);
    else return (float)static_cast<const _Float16*>(a.bias)[o];
}

// accumulators begin with the bias of their output (in LDS: the wave's first output's on), or with zero
template <bool DX, int TO, int TP> __device__ __forceinline__ void begin(f32x16 (&acc)[TO][TP], const float* bias, int lane) {
#pragma unroll
    for (int i = 0; i < TO; ++i) {
        f32x16 b = {0};
        if (!DX)
#pragma unroll
            for (int r = 0; r < 16; ++r) b[r] = bias[32 * i + (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5)];
#pragma unroll
        for (int k = 0; k < TP; ++k) acc[i][k] = b;
    }
}

// ------------------------------------------------------------------------------------------------------------------------------ Y = act(A B + bias)
// One workgroup = BP rows x BO outputs, 4 waves of (BP / 2) x (BO / 2); D[output][row] so that a lane's accumulators are runs of 4 outputs of ONE row.  The reduction runs
// in steps of BK staged through LDS: the next step's elements travel into registers while this step's products run.
// Neighbouring workgroups of one XCD take the output tiles of the same rows (the rows are read from HBM once and then from that XCD's L2).  float32 is bound by the six products
// and their operands' splitting and staging: 64 064 x 384 -> 384 121 us (156 TFLOP/s of float32, 936 of products: matrix cores busy 42 %, vector units 37 %; a library's largest
// bfloat16 product reaches 1 155 to 1 320, its float32 product of 786 432 rows 132), its input gradient 126 for 65 536 rows.
template <int T, bool DX, int BP, int BO>
__global__ __launch_bounds__(256, 2) void k_dense_rows(DenseRows a) {
    constexpr int PARTS = T == LT_F32 ? 3 : 1, BK = T == LT_F32 ? 32 : 64;
    constexpr int TP = BP / 64, TO = BO / 64;                      // 32-wide tiles of a wave
    constexpr int XC = BP * BK / 8 / 256, WC = BO * BK / 8 / 256;  // 8-element chunks a thread stages
    constexpr int XPLANE = BP * BK, WPLANE = BO * BK;
    constexpr int STAGE = PARTS * (XPLANE + WPLANE) * 2, OUT = 4 * Window<TO, T>::bytes;
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
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wp = (wave >> 1) * (BP / 2), wo = (wave & 1) * (BO / 2);
    if (!DX && t < BO) bias[t] = bias_at<T>(a, o0 + t);

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
            else stage8<T>(wt + across<BO>(c / (BO / 8), (c % (BO / 8)) >> 2) + 8 * (c & 3), WPLANE, wr[i]);
        }
    };

    f32x16 acc[TO][TP];
    load(0);
    for (int k0 = 0; k0 < a.r; k0 += BK) {
        if (k0) __syncthreads();
        stage();
        __syncthreads();
        if (k0 == 0) begin<DX>(acc, bias + wo, lane);
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
                    w[q] = DX ? frag_across<BO>(wt + q * WPLANE, (wo >> 5) + i, ks, lane) : frag_along<BK>(wt + q * WPLANE, wo + 32 * i, ks, lane);
#pragma unroll
                for (int k = 0; k < TP; ++k) acc[i][k] = product<T, PARTS, PARTS>(w, x[k], acc[i][k]);
            }
        }
    }
    __syncthreads();

    write_rows<T, DX, TO, TP>(a, acc, lds + wave * Window<TO, T>::bytes, p0 + wp, o0 + wo, lane);
}

// outputs o .. o + 7 of row p, and their codes (four neighbouring lanes hold a block; rows and outputs beyond the last are not written)
template <int T, bool DX> __device__ __forceinline__ void finish8(const DenseRows& a, long p, int o, const float (&f)[8]) {
    const Raw8<T> v = from_floats<T>(f);
    const bool in = p < a.n;
    if (in && o < a.o) store8<T>(static_cast<char*>(a.y) + p * a.ldy * Bytes<T>::v, o, a.o, v);
    if (!DX && a.codes) {
        u32x2 codes; unsigned scale;
        encode8<T>(v, a.is_signed != 0, codes, scale);
        const int o32 = (a.o + 31) & ~31;
        if (in) {
            *reinterpret_cast<u32x2*>(a.codes + p * o32 + o) = codes;
            if ((o & 31) == 0) a.scales[p * (o32 >> 5) + (o >> 5)] = (uint8_t)scale;
        }
    }
}

// The form for few rows, where one latency after the other is what a call costs: a workgroup makes 32 rows x 32 outputs, each of its 4 waves over a quarter of the reduction, straight
// from global memory (operands in the order they lie there, 4 steps asked for at once), and the quarters meet in LDS once.  1 x 512 -> 512 bfloat16: 5.0 us of kernel.
constexpr int FEW_ROW = 36, FEW_LDS = 4 * 32 * FEW_ROW;      // floats
template <int T, bool DX> __device__ __forceinline__ void dense_few(const DenseRows& a, unsigned block, float* sums) {
    constexpr int U = 4, RS = FEW_ROW;
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), i = lane & 31, h = lane >> 5;
    const int ot = (a.o + 31) >> 5, o0 = (int)(block % ot) * 32;
    const long p0 = (long)(block / ot) * 32;
    const int steps = (a.r + 15) >> 4, quarter = (steps + 3) >> 2, s1 = min(steps, (wave + 1) * quarter), r32 = (a.r + 31) & ~31;
    const long p = min(p0 + i, a.n - 1);                 // (rows and outputs beyond the last: the last again, not written)
    const int o = min(o0 + i, a.o - 1);
    const char* x = static_cast<const char*>(a.a) + p * a.lda * Bytes<T>::v;
    const char* w = static_cast<const char*>(a.w) + (DX ? (long)o : o * a.ldw) * Bytes<T>::v;
    const bool whole = (a.r & 7) == 0;                   // every 8-element chunk of the reduction is whole or absent
    f32x16 acc = {0};
    for (int s0 = wave * quarter; s0 < s1; s0 += U) {
        Raw8<T> xv[U], wv[U];
        u32x2 q[U];
        if (whole) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = min(16 * (s0 + u) + 8 * h, a.r - 8);
                xv[u].q[0] = load16(x + (long)k * Bytes<T>::v);
                if constexpr (T == LT_F32) xv[u].q[1] = load16(x + (long)k * 4 + 16);
                q[u] = u32x2{0x01010101u, 0x01010101u};
                if (DX && a.open) q[u] = *reinterpret_cast<const u32x2*>(a.open + p * r32 + k);
                if (!DX) {
                    wv[u].q[0] = load16(w + (long)k * Bytes<T>::v);
                    if constexpr (T == LT_F32) wv[u].q[1] = load16(w + (long)k * 4 + 16);
                } else {
                    wv[u] = zero8<T>();
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        if constexpr (T == LT_F32) wv[u].q[e >> 2][e & 3] = *reinterpret_cast<const unsigned*>(w + (k + e) * a.ldw * 4);
                        else wv[u].q[0][e >> 1] |= (unsigned)*reinterpret_cast<const unsigned short*>(w + (k + e) * a.ldw * 2) << (16 * (e & 1));
                    }
                }
            }
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = 16 * (s0 + u) + 8 * h;
                xv[u] = load8<T>(x, k, a.r);
                q[u] = u32x2{0x01010101u, 0x01010101u};
                if (DX && a.open && k < r32) q[u] = *reinterpret_cast<const u32x2*>(a.open + p * r32 + k);
                if (!DX) {
                    wv[u] = load8<T>(w, k, a.r);
                } else {
                    wv[u] = zero8<T>();
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (k + e < a.r) {
                            if constexpr (T == LT_F32) wv[u].q[e >> 2][e & 3] = *reinterpret_cast<const unsigned*>(w + (k + e) * a.ldw * 4);
                            else wv[u].q[0][e >> 1] |= (unsigned)*reinterpret_cast<const unsigned short*>(w + (k + e) * a.ldw * 2) << (16 * (e & 1));
                        }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s0 + u >= s1) break;
            if (DX) close8<T>(xv[u], q[u]);
            if (16 * (s0 + u) + 8 * h >= a.r) xv[u] = wv[u] = zero8<T>();
            u32x4 xp[Parts<T>::n], wp[Parts<T>::n];
            parts_of<T>(xv[u], xp);
            parts_of<T>(wv[u], wp);
            acc = product<T, Parts<T>::n, Parts<T>::n>(wp, xp, acc);
        }
    }
#pragma unroll
    for (int g = 0; g < 4; ++g)
        *reinterpret_cast<u32x4*>(sums + (wave * 32 + i) * RS + 8 * g + 4 * h) = u32x4{as_bits(acc[4 * g]), as_bits(acc[4 * g + 1]), as_bits(acc[4 * g + 2]), as_bits(acc[4 * g + 3])};
    __syncthreads();
    if (t >= 128) return;
    const int row = t >> 2, c = 8 * (t & 3);
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float v = DX ? 0.0f : bias_at<T>(a, o0 + c + e);
#pragma unroll
        for (int q = 0; q < 4; ++q) v += sums[(q * 32 + row) * RS + c + e];
        if (!DX && a.relu) v = __builtin_elementwise_maximum(v, 0.0f);
        f[e] = !DX && o0 + c + e >= a.o ? 0.0f : v;      // (columns beyond the layer's outputs are coded 0)
    }
    finish8<T, DX>(a, p0 + row, o0 + c, f);
}

template <int T, bool DX> __global__ __launch_bounds__(256) void k_dense_few(DenseRows a) {
    __shared__ __attribute__((aligned(16))) float sums[FEW_LDS];
    dense_few<T, DX>(a, blockIdx.x, sums);
}

// One lane's 8 reduction elements of output i of the weights, zeros beyond the layer (16-bit types)
template <int T, bool DX> __device__ __forceinline__ u32x4 weight_fragment(const DenseRows& a, int i, int r0) {
    u32x4 v = {0, 0, 0, 0};
    if (i < a.o) {
        if (!DX) {
            v = load8<T>(static_cast<const char*>(a.w) + (long)i * a.ldw * 2, r0, a.r).q[0];
        } else {
            const unsigned short* w = static_cast<const unsigned short*>(a.w) + i;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (r0 + e < a.r) v[e >> 1] |= (unsigned)w[(long)(r0 + e) * a.ldw] << (16 * (e & 1));
        }
    }
    return v;
}

// The form for many rows of at most 32 outputs (16-bit types): a wave takes 32 rows at a time, straight from memory in the order the matrix instruction wants them; the weights'
// operands stay in LDS.  Chunks are read whole: what lies behind a row's end is cleared in registers, and only rows with 7 more behind them are read so.  Bound by HBM once rows
// are long (100 000 x 500 -> 32 bfloat16: 34 us, 3.1 TB/s), by the many small stores where they are short (730 935 x 26 -> 5: 15 us, 3 TB/s).
template <int T, bool DX> __global__ __launch_bounds__(256, 4) void k_dense_narrow(DenseRows a) {
    constexpr int U = 4;
    extern __shared__ __attribute__((aligned(16))) float narrow[];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), i = lane & 31, h = lane >> 5;
    const int steps = (a.r + 15) >> 4, r32 = (a.r + 31) & ~31, last = (a.r - 1) & ~7;
    float* win = narrow + wave * 32 * FEW_ROW;
    u32x4* wf = reinterpret_cast<u32x4*>(narrow + FEW_LDS);
    for (int id = t; id < 64 * steps; id += 256) wf[id] = weight_fragment<T, DX>(a, id & 31, 16 * (id >> 6) + 8 * ((id >> 5) & 1));
    f32x16 bias = {0};
    if (!DX)
#pragma unroll
        for (int r = 0; r < 16; ++r) bias[r] = bias_at<T>(a, (r & 3) + 8 * (r >> 2) + 4 * h);
    __syncthreads();
    for (long p0 = 32 * ((long)blockIdx.x * 4 + wave); p0 < a.n; p0 += 128L * gridDim.x) {
        const long p = min(p0 + i, a.n - 1);
        const char* x = static_cast<const char*>(a.a) + p * a.lda * 2;
        const bool all = p0 + 32 + 7 <= a.n;
        f32x16 acc = bias;
        for (int s0 = 0; s0 < steps; s0 += U) {
            Raw8<T> xv[U];
            u32x2 q[U];
            if (all) {
#pragma unroll
                for (int u = 0; u < U; ++u) xv[u].q[0] = load16(x + 2L * min(16 * (s0 + u) + 8 * h, last));
            } else {
#pragma unroll
                for (int u = 0; u < U; ++u) xv[u] = load8<T>(x, 16 * (s0 + u) + 8 * h, a.r);
            }
            if (DX && a.open)
#pragma unroll
                for (int u = 0; u < U; ++u) q[u] = *reinterpret_cast<const u32x2*>(a.open + p * r32 + min(16 * (s0 + u) + 8 * h, last));
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (s0 + u >= steps) break;
                if (DX && a.open) close8<T>(xv[u], q[u]);
                if (16 * (s0 + u) + 16 > a.r) {
                    const int left = a.r - 16 * (s0 + u) - 8 * h;
#pragma unroll
                    for (int j = 0; j < 4; ++j) xv[u].q[0][j] = left >= 2 * j + 2 ? xv[u].q[0][j] : left == 2 * j + 1 ? xv[u].q[0][j] & 0xffffu : 0u;
                }
                acc = mfma<T>(wf[64 * (s0 + u) + lane], xv[u].q[0], acc);
            }
        }
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<u32x4*>(win + i * FEW_ROW + 8 * g + 4 * h) = u32x4{as_bits(acc[4 * g]), as_bits(acc[4 * g + 1]), as_bits(acc[4 * g + 2]), as_bits(acc[4 * g + 3])};
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            const int row = 16 * z + (lane >> 2), c = 8 * (lane & 3);
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float v = win[row * FEW_ROW + c + e];
                f[e] = !DX && c + e >= a.o ? 0.0f : !DX && a.relu ? __builtin_elementwise_maximum(v, 0.0f) : v;
            }
            finish8<T, DX>(a, p0 + row, c, f);
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// The weights as matrix operands for k_dense_tall: [32-wide tile][16 reduction elements][lane][8], zeros beyond the layer
template <int T, bool DX> __global__ __launch_bounds__(256) void k_dense_fragments(DenseRows a, u32x4* wf, int tiles, int steps) {
    const int id = blockIdx.x * 256 + threadIdx.x;
    const int lane = id & 63, ks = (id >> 6) % steps, tile = (id >> 6) / steps;
    if (tile >= tiles) return;
    wf[id] = weight_fragment<T, DX>(a, 32 * tile + (lane & 31), 16 * ks + 8 * (lane >> 5));
}

constexpr int TALL_ROWS = 128;
// eight 16-bit elements moved down by `n` (0 or less: not at all; 8 or more: nothing is left), zeros behind them
__device__ __forceinline__ u32x4 drop16(u32x4 v, int n) {
    unsigned long long lo = v[0] | (unsigned long long)v[1] << 32, hi = v[2] | (unsigned long long)v[3] << 32;
    const int s = 16 * max(n, 0);
    const unsigned long long l = s == 0 ? lo : s < 64 ? lo >> s | hi << (64 - s) : s < 128 ? hi >> (s - 64) : 0, u = s < 64 ? hi >> s : 0;
    return u32x4{(unsigned)l, (unsigned)(l >> 32), (unsigned)u, (unsigned)(u >> 32)};
}
// place of the 16-byte chunk c of a row of CH chunks: 16 rows x one chunk fall on all banks
template <int CH> __device__ __forceinline__ int tall_at(int row, int c) { return (row * CH + (c ^ (CH == 8 ? (row >> 1) & 7 : row & 15))) * 8; }

// What k_dense_tall makes: the input gradient, or Y alone, or Y with its checkpoint behind a ReLU / without one
enum TallMode { TALL_DX = 0, TALL_Y = 1, TALL_RELU_KEEP = 2, TALL_KEEP = 3 };

// 32 rows x 64 outputs of Y from their accumulators.  A lane has outputs (r & 3) + 8 (r >> 2) + 4 h of row i; halves of the wave swap packed pairs so that it holds 16 neighbouring
// outputs (16 h on): the block's largest value is one more swap away, 16 codes are one 16-byte word.  Everything leaves through `win` (2.5 KB of LDS for each wave) in
// pieces of 64 bytes of a row: the address unit takes one such piece a cycle, and 16 bytes of 64 rows cost it 64 cycles where 64 bytes of 16 rows cost 16 (stored straight
// from the lanes, results and codes took 270 us more for 786 432 x 512).
struct Out { char* y; uint8_t* codes; uint8_t* scales; long ldy; int o32, rows, o; };      // at the first row and output; rows that are there, outputs from the first on
template <int T, int MODE> __device__ __forceinline__ void write_rows64(const DenseRows& a, const f32x16& a0, const f32x16& a1, const Out& out, int lane, char* win) {
    constexpr bool KEEP = MODE == TALL_RELU_KEEP || MODE == TALL_KEEP, SIGNED = MODE == TALL_KEEP;
    constexpr int RS = 80;      // bytes of a row in the window (64 and a step to the next banks)
    const int h = lane >> 5, i = lane & 31;
    u32x4 c[2];
    unsigned scales = 0;
#pragma unroll
    for (int tile = 0; tile < 2; ++tile) {
        const f32x16& acc = tile ? a1 : a0;
        unsigned d[4][2];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = acc[4 * g + e];
                if (MODE == TALL_RELU_KEEP || (MODE == TALL_Y && a.relu)) v[e] = __builtin_elementwise_maximum(v[e], 0.0f);      // (a NaN stays, -0 becomes 0)
            }
            d[g][0] = pack2<T>(v[0], v[1]);
            d[g][1] = pack2<T>(v[2], v[3]);
        }
        Raw8<T> half[2];
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const auto s = __builtin_amdgcn_permlane32_swap(d[g][j], d[g + 2][j], false, false);
                half[g].q[0][j] = s[0];
                half[g].q[0][2 + j] = s[1];
            }
        char* mine = win + i * RS + 32 * h;
        *reinterpret_cast<u32x4*>(mine) = half[0].q[0];
        *reinterpret_cast<u32x4*>(mine + 16) = half[1].q[0];
        if (KEEP) {
            const int have = out.o - 32 * tile - 16 * h;
            if (out.o < 64)      // (columns beyond the layer's outputs are coded 0)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (e >= have) half[e >> 3].q[0][(e & 7) >> 1] &= (e & 1) ? 0x0000ffffu : 0xffff0000u;
            u16x2 m = {0, 0};      // magnitudes as integers; behind a ReLU there is no sign: the bits themselves (a NaN's with it)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const unsigned u = half[e >> 2].q[0][e & 3] & (SIGNED ? 0x7fff7fffu : 0xffffffffu);
                m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, u));
            }
            Block b;
            b.mag = max((unsigned)m[0], (unsigned)m[1]);
            const auto s = __builtin_amdgcn_permlane32_swap(b.mag, b.mag, false, false);
            b.mag = b.top = max(s[0], s[1]);
            const Step st = step_of<T>(b, SIGNED);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const u32x2 q = codes_of<T>(half[e], st, SIGNED);
                c[tile][2 * e] = q[0];
                c[tile][2 * e + 1] = q[1];
            }
            scales |= st.scale << (8 * tile);
        }
        __builtin_amdgcn_wave_barrier();
        const int o = 32 * tile + 8 * (lane & 3);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int row = 16 * j + (lane >> 2);
            Raw8<T> v;
            v.q[0] = *reinterpret_cast<const u32x4*>(win + row * RS + 16 * (lane & 3));
            char* y = out.y + row * out.ldy;
            if (out.o >= 64) {
                if (row < out.rows) __builtin_memcpy(y + 2 * o, &v.q[0], 16);
            } else if (row < out.rows) store8<T>(y, o, out.o, v);
        }
        __builtin_amdgcn_wave_barrier();
    }
    if (KEEP) {
#pragma unroll
        for (int tile = 0; tile < 2; ++tile) *reinterpret_cast<u32x4*>(win + i * RS + 32 * tile + 16 * h) = c[tile];
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int row = 16 * j + (lane >> 2), o = 16 * (lane & 3);
            const u32x4 v = *reinterpret_cast<const u32x4*>(win + row * RS + o);
            if (row < out.rows && o < ((out.o + 31) & ~31)) __builtin_memcpy(out.codes + row * out.o32 + o, &v, 16);
        }
        if (h == 0 && i < out.rows) {
            uint8_t* s = out.scales + i * (out.o32 >> 5);
            s[0] = (uint8_t)scales;
            if (out.o > 32) s[1] = (uint8_t)(scales >> 8);
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// The 16-bit types' form for many rows.  No unit is full: for 786 432 x 512 -> 512 with the checkpoint the address units (see write_rows64) are busy 58 % of the time, the matrix cores
// 29 %, HBM carries 3.0 TB/s, and the waves wait a third of their time (as the input gradient: 63 %, 32 %, 3.9 TB/s).  Two workgroups stay on each compute unit (one beyond 6 passes) and
// flow through their work, 128 rows x 256 outputs at a time: while a piece of the rows
// (128 x COLS columns) is multiplied out of one LDS buffer, the next one — the next work item's first, too — is on its way in registers, goes to the other buffer, and the
// piece after that is asked for before results are written; the other workgroup multiplies meanwhile.  A wave takes 128 rows x 64 outputs, so a fragment of the rows is
// read once from LDS for each wave, and a fragment of the weights once from L2 for the workgroup.  Items of the same rows are neighbours on one XCD.  COLS: 128, or 64 for
// layers that read no more.  786 432 x 512 x 512 bfloat16: 700 us with the checkpoint (2.1 GB: 3.0 TB/s), 570 us without, 630 us as the input gradient.  Tried and slower:
// steps of 64 columns with one step under way (940 us); all columns of 64 rows at once, the weights read twice as often (750); weights kept in LDS and rows straight to
// registers as operands (915: 16 bytes of 32 rows a load, address units full).
template <int T, int MODE, int COLS>
__global__ __launch_bounds__(256, 2) void k_dense_tall(DenseRows a, const u32x4* wf, int passes) {
    constexpr bool DX = MODE == TALL_DX;
    constexpr int TP = 4, TO = 2, AHEAD = 2, BO = 256, NT = 256, CH = COLS / 8, RP = NT / CH, NC = TALL_ROWS / RP, BUFFER = TALL_ROWS * COLS;
    extern __shared__ __attribute__((aligned(16))) unsigned short lds[];
    char* wins = reinterpret_cast<char*>(lds + 2 * BUFFER);
    float* bias = reinterpret_cast<float*>(wins + 4 * 2560);
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int steps = (a.r + 63) / 64 * 4, pieces = (a.r + COLS - 1) / COLS, r32 = (a.r + 31) & ~31, o32 = (a.o + 31) & ~31;
    if (!DX) for (int i = t; i < passes * BO; i += NT) bias[i] = bias_at<T>(a, i);
    // work item j of XCD x: rows of tile x + 8 (j / passes), outputs of pass j % passes; a workgroup takes every (gridDim / 8)-th
    const long tiles = (a.n + TALL_ROWS - 1) / TALL_ROWS;
    const int xcd = blockIdx.x & 7, first_item = blockIdx.x >> 3, stride_item = gridDim.x >> 3;
    const long items = xcd < tiles ? (tiles - xcd + 7) / 8 * passes : 0;
    const long mine = first_item < items ? (items - first_item + stride_item - 1) / stride_item : 0, count = mine * pieces;

    // where the sequence of pieces stands: the loads run ahead of the products
    struct At { long tile; int pass, piece; };
    auto next = [&](At& x) {
        if (++x.piece == pieces) {
            x.piece = 0;
            x.pass += stride_item;
            x.tile += 8 * (x.pass / passes);
            x.pass %= passes;
        }
    };
    // the thread's 16-byte chunk of every RP-th row of a piece.  Rows behind the last are the last again (their results are not written), a chunk that hangs over the row's end is read
    // from 8 elements before it and moved (stage): no branches, the loads travel together
    const int row = t / CH, col = 8 * (t % CH);
    const long stride = a.lda * 2;
    unsigned short* place = lds + tall_at<CH>(row, t % CH);
    Raw8<T> v[NC];
    u32x2 q[NC];
    int held = 0;      // the piece that the registers hold
    auto load = [&](const At& x) {
        const long p0 = x.tile * TALL_ROWS;
        const int k = x.piece * COLS + col, last = (int)min(a.n - 1 - p0, (long)(TALL_ROWS - 1));
        const char* base = static_cast<const char*>(a.a) + p0 * stride;
        const unsigned at = 2 * min(k, a.r - 8);
        held = x.piece;
#pragma unroll
        for (int i = 0; i < NC; ++i) v[i].q[0] = load16(base + ((unsigned)min(row + i * RP, last) * (unsigned)stride + at));
        if (DX && a.open) {
            const uint8_t* open = a.open + p0 * r32;
            const unsigned at8 = min(k, r32 - 8);
#pragma unroll
            for (int i = 0; i < NC; ++i) q[i] = *reinterpret_cast<const u32x2*>(open + ((unsigned)min(row + i * RP, last) * (unsigned)r32 + at8));
        }
    };
    auto stage = [&](int b) {
        if ((held + 1) * COLS > a.r) {      // the row ends in this piece
            const int over = held * COLS + col - (a.r - 8);      // elements that the chunk was read too early by; 8 and more: nothing of it is in the row
#pragma unroll
            for (int i = 0; i < NC; ++i) v[i].q[0] = drop16(v[i].q[0], over);
        }
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            if (DX && a.open) close8<T>(v[i], q[i]);
            *reinterpret_cast<u32x4*>(place + b * BUFFER + i * RP * COLS) = v[i].q[0];
        }
    };

    f32x16 acc[TO][TP];
    At in{xcd + 8 * (long)(first_item / passes), first_item % passes, 0}, now = in;
    const int frow = lane & 31, fx = CH == 8 ? (frow >> 1) & 7 : frow & 15;      // a fragment's row in its 32, what its chunks are crossed with
    const unsigned wlane = 16 * lane;
    // The weights' fragments are one stream over all pieces, AHEAD steps in front of the products: loads come back in the order they were asked for, so a piece's first fragments
    // are asked for before the rows of the piece after it — behind those they would wait for HBM
    u32x4 w[AHEAD][TO];
    auto weights_of = [&](const At& x) { return reinterpret_cast<const char*>(wf) + ((size_t)(x.pass * (BO / 32) + wave * TO) * steps + x.piece * (COLS / 16)) * 1024; };
    auto weights = [&](const char* wl, int step, u32x4 (&to)[TO]) {
#pragma unroll
        for (int i = 0; i < TO; ++i) to[i] = *reinterpret_cast<const u32x4*>(wl + (size_t)(i * steps + step) * 1024 + wlane);
    };
    if (count > 0) {
        load(in);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) weights(weights_of(in), u, w[u]);
        next(in);
        stage(0);
    }
    if (count > 1) { load(in); next(in); }
    __syncthreads();
    for (long s = 0; s < count; ++s) {
        const int b = (int)s & 1, o0 = now.pass * BO + wave * 64, size = min(steps - now.piece * (COLS / 16), COLS / 16);
        const char* wl = weights_of(now);
        At after = now;
        if (s + 1 < count) next(after);
        const char* wn = weights_of(after);
        asm volatile("" ::: "memory");      // (the bias and the weights of a one-piece layer are the same in every round: kept in registers they spill)
        if (now.piece == 0) begin<DX>(acc, bias + o0, lane);
        const unsigned short* x0 = lds + b * BUFFER + frow * COLS;
        auto rows_at = [&](int step, u32x4 (&x)[TP]) {
            const unsigned short* xs = x0 + (((2 * step + (lane >> 5)) ^ fx) * 8);
#pragma unroll
            for (int k = 0; k < TP; ++k) x[k] = *reinterpret_cast<const u32x4*>(xs + 32 * k * COLS);
        };
        u32x4 x[2][TP];
        rows_at(0, x[0]);
#pragma unroll 1
        for (int s0 = 0; s0 < size; s0 += AHEAD) {      // (a multiple of 4)
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int st = s0 + u;
                rows_at(st + 1 < size ? st + 1 : st, x[(u + 1) & 1]);       // (the last ones again: no branch)
#pragma unroll
                for (int i = 0; i < TO; ++i)
#pragma unroll
                    for (int k = 0; k < TP; ++k) acc[i][k] = mfma<T>(w[u][i], x[u & 1][k], acc[i][k]);
                const bool here = st + AHEAD < size;
                weights(here ? wl : wn, here ? st + AHEAD : st + AHEAD - size, w[u]);
                __builtin_amdgcn_sched_barrier(0);      // (left alone, the compiler moves these loads down to their use)
            }
        }
        if (s + 1 < count) stage(b ^ 1);
        if (s + 2 < count) { load(in); next(in); }
        if (now.piece == pieces - 1 && o0 < a.o) {
            const long p0 = now.tile * TALL_ROWS;
#pragma unroll
            for (int k = 0; k < TP; ++k) {
                const long p = p0 + 32 * k;
                const Out out{static_cast<char*>(a.y) + (p * a.ldy + o0) * 2, a.codes + p * o32 + o0, a.scales + p * (o32 >> 5) + (o0 >> 5), 2 * a.ldy, o32, (int)min(a.n - p, 32L), a.o - o0};
                write_rows64<T, MODE>(a, acc[0][k], acc[1][k], out, lane, wins + 2560 * wave);
            }
        }
        now = after;
        __syncthreads();
    }
}

// --------------------------------------------------------------------------------------------------------------------------------- dW = dZ^T X, db
// One workgroup = a tile of WO outputs x WK input columns over its piece of the rows, BR rows a step.  Both operands lie with the REDUCTION index as the row, as
// they do in memory, and are turned by the transposing LDS read.  The pieces' sums go to `part` and are added in order by k_dense_weights_sum: no atomics, the same
// bits every time.
//
// 128 x 128: 4 waves of 64 x 64, two workgroups on a compute unit; 256 x 256: 16 waves, half as many reads of either operand; 32 on the side of a narrow layer: a wave has one
// 32 x 32 tile, or a share of the rows of the only one.  786 432 x 512 -> 512 float16: 545 us (1.7 GB: 3.2 TB/s; 760 TFLOP/s), on the way through registers and LDS that
// turns and decodes the operands (vector units busy 45 % of the time, address units 44 %, matrix cores 38 %, LDS 29 %; the waves wait 42 % of theirs); 65 536 x 384 float32 86 us (41, 29,
// 27, 18); 196 608 x 512 -> 4 float32 52.
template <int T, int WO, int WK> struct WeightsTile {
    static constexpr int NT = WO == 256 ? 1024 : 256, PARTS = T == LT_F32 ? 3 : 1, BR = T == LT_F32 && WO != 32 ? 32 : 64;
    static constexpr int ZPLANE = BR * WO, XPLANE = BR * WK, BUFFER = PARTS * ZPLANE + XPLANE;
    static constexpr int TO = WO >= 128 && WK >= 128 ? 2 : 1, TK = TO;                       // 32-wide tiles of a wave
    static constexpr int SHARE = NT / 64 / ((WO / 32 / TO) * (WK / 32 / TK));                // waves that share a tile, each with every SHARE-th 16 rows
};
template <int T, int WO, int WK> __device__ __forceinline__ void dense_weights_tile(const DenseWeights& a, unsigned block, unsigned short* lds) {
    using W = WeightsTile<T, WO, WK>;
    constexpr int PARTS = W::PARTS, BR = W::BR, NT = W::NT, TO = W::TO, TK = W::TK, ZPLANE = W::ZPLANE, BUFFER = W::BUFFER, SHARE = W::SHARE;
    // threads a row of either tile, rows at a time, 8-column chunks a thread stages (a thread without one stages another's again)
    constexpr int RTZ = WO / 8, RTX = WK / 8, RPZ = NT / RTZ < BR ? NT / RTZ : BR, RPX = NT / RTX < BR ? NT / RTX : BR, NZ = BR / RPZ, NX = BR / RPX, NC = NZ > NX ? NZ : NX;
    static_assert(NC <= BR / 16, "a chunk for each step of 16 rows at most");
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int kt = (a.k + WK - 1) / WK, ot = (a.o + WO - 1) / WO, tiles = kt * ot;
    const long j = block >> 3;
    const int split = (int)(j / tiles) * 8 + (block & 7);
    if (split >= a.splits) return;
    const int tile = (int)(j % tiles), k0 = (tile % kt) * WK, o0 = (tile / kt) * WO;
    const long steps = (a.n + BR - 1) / BR;
    const long s0 = steps * split / a.splits, s1 = steps * (split + 1) / a.splits;
    const int k32 = (a.k + 31) & ~31, o32 = (a.o + 31) & ~31;
    // the thread's 8 columns of either tile are the same in every step; its rows: zrow + RPZ * i, xrow + RPX * i.  Addresses are a scalar base that moves with the steps and 32-bit
    // offsets
    const int zcc = 8 * (t % RTZ), zrow = (t / RTZ) % BR, xcc = 8 * (t % RTX), xrow = (t / RTX) % BR;
    // (columns beyond the outputs or inputs: any, their sums are not written)
    const int zc = o0 + zcc < a.o ? o0 + zcc : 0, xc0 = k0 + xcc < k32 ? k0 + xcc : 0;
    const unsigned zo = (unsigned)(zrow * (int)a.lddy + zc) * Bytes<T>::v, oo = zrow * o32 + zc, co = xrow * k32 + xc0, so = xrow * (k32 >> 5) + (xc0 >> 5);
    const char* zb = static_cast<const char*>(a.dy) + s0 * BR * a.lddy * Bytes<T>::v;
    const uint8_t *ob = a.open + s0 * BR * o32, *cb = a.x.codes + s0 * BR * k32, *sb = a.x.scales + s0 * BR * (k32 >> 5);
    const long rows = a.n - s0 * BR;

    Raw8<T> zr[NZ];
    u32x2 cr[NZ], xc[NX];
    unsigned xs[NX];
    // Chunk i of a step (counted from s0) into registers.  ALL: every row of the step is there and 7 more behind it, so that whole chunks may be read beyond a row's last column
    // (their sums are not written): straight code, the loads travel together.  Otherwise what is there, and zeros.
    auto load = [&](long step, int i, auto ALL) {
        if (i < NZ) {
            const long at = step * BR + RPZ * i;
            const char* z = zb + at * a.lddy * Bytes<T>::v;
            const uint8_t* open = ob + at * o32;
            if constexpr (decltype(ALL)::value) {
                zr[i].q[0] = load16(z + zo);
                if constexpr (T == LT_F32) zr[i].q[1] = load16(z + zo + 16);
                if (a.open) cr[i] = *reinterpret_cast<const u32x2*>(open + oo);
            } else {
                const bool in = at + zrow < rows;
                zr[i] = in ? load8<T>(z + zo, 0, a.o - zc) : zero8<T>();
                if (a.open && in) cr[i] = *reinterpret_cast<const u32x2*>(open + oo);
            }
        }
        if (i < NX) {
            const long at = step * BR + RPX * i;
            const uint8_t *codes = cb + at * k32, *scales = sb + at * (k32 >> 5);
            const bool in = decltype(ALL)::value || at + xrow < rows;
            xc[i] = in ? *reinterpret_cast<const u32x2*>(codes + co) : u32x2{0, 0};
            xs[i] = in ? scales[so] : 127u;
        }
    };
    auto stage = [&](unsigned short* zt, int i) {
        if (i < NZ) {
            if (a.open) close8<T>(zr[i], cr[i]);
            stage8<T>(zt + across<WO>(zrow + RPZ * i, (t % RTZ) >> 2) + 8 * (t & 3), ZPLANE, zr[i]);
        }
        if (i < NX) {
            unsigned short* to = zt + PARTS * ZPLANE + across<WK>(xrow + RPX * i, (t % RTX) >> 2) + 8 * (t & 3);
            auto put = [&](const float (&f)[8]) {
                u32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e)      // a value has at most 8 significant bits: its upper 16 bits are all of it
                    v[e] = T == LT_F16 ? pack2<LT_F16>(f[2 * e], f[2 * e + 1]) : __builtin_amdgcn_perm(as_bits(f[2 * e + 1]), as_bits(f[2 * e]), 0x07060302u);
                *reinterpret_cast<u32x4*>(to) = v;
            };
            float f[8];
            decode8(xc[i], xs[i], a.x.is_signed != 0, f);
            put(f);
            if (__builtin_expect(large_block<T>(xs[i]), 0)) {      // written again, out of the way: 786 432 x 512 float16 takes 5 % longer where the compiler weighs both alike
                decode8_large<T>(xc[i], xs[i], a.x.is_signed != 0, f);
                put(f);
            }
        }
    };

    const int place = wave / SHARE, wo = (place / (WK / 32 / TK)) * TO, wk = (place % (WK / 32 / TK)) * TK;      // the wave's first 32-wide tile of either side
    f32x16 acc[TO][TK];
#pragma unroll
    for (int i = 0; i < TO; ++i)
#pragma unroll
        for (int k = 0; k < TK; ++k) acc[i][k] = f32x16{0};
    // The bias gradient falls off the fragments (a lane has 8 rows of one output).  It is one sum over all rows with nothing to average an error out: added up in 64 bits, which is as
    // much work as products are, so it is dealt out — a wave's first 32 outputs to the workgroups of the first column tile, the next to those of the second, and 16 rows in
    // turn to the waves of one row of tiles (one wave of one workgroup for all of it: 786 432 x 512 took 650 us instead of 590)
    constexpr int TURNS = WK / 32 / TK;
    const int turn = place % TURNS;
    auto sums = [&](int i) { return a.db != nullptr && (kt > 1 ? i : 0) * WK == k0; };
    double bs[TO] = {};
    auto multiply = [&](const unsigned short* zt, int ks) {
        if (SHARE > 1 && ks % SHARE != wave % SHARE) return;
        const unsigned short* xt = zt + PARTS * ZPLANE;
        u32x4 x[TK][1];
#pragma unroll
        for (int k = 0; k < TK; ++k) x[k][0] = frag_across<WK>(xt, wk + k, ks, lane);
#pragma unroll
        for (int i = 0; i < TO; ++i) {
            u32x4 z[PARTS];
#pragma unroll
            for (int q = 0; q < PARTS; ++q) z[q] = frag_across<WO>(zt + q * ZPLANE, wo + i, ks, lane);
#pragma unroll
            for (int k = 0; k < TK; ++k) acc[i][k] = product<T, PARTS, 1>(z, x[k], acc[i][k]);
            if (sums(i) && ks % TURNS == turn)
#pragma unroll
                for (int q = 0; q < PARTS; ++q) {
                    Raw8<T == LT_F16 ? LT_F16 : LT_BF16> v;
                    v.q[0] = z[q];
                    float f[8];
                    to_floats<T == LT_F16 ? LT_F16 : LT_BF16>(v, f);
                    bs[i] += (double)(((f[0] + f[1]) + (f[2] + f[3])) + ((f[4] + f[5]) + (f[6] + f[7])));
                }
        }
    };
    // One barrier a step: while a step's products run, the next one's elements — already in registers — are masked, decoded and written to the other buffer, a chunk between
    // 16 rows of products and the next, and the chunk's registers are asked for the step after that: a load has a whole step to arrive
    const long count = s1 - s0;
    constexpr std::true_type all{};
    constexpr std::false_type some{};
    if (count > 0) {
        if (rows >= 2 * BR + 7 && count > 1) {
#pragma unroll
            for (int i = 0; i < NC; ++i) load(0, i, all);
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                stage(lds, i);
                load(1, i, all);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NC; ++i) load(0, i, some);
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                stage(lds, i);
                if (count > 1) load(1, i, some);
            }
        }
        __syncthreads();
        long s = 0;
        const long full = (rows - 7) / BR - 2;      // steps whose next but one is whole
        for (; s + 2 < count && s < full; ++s) {
            const int b = (int)s & 1;
#pragma unroll
            for (int i = 0; i < BR / 16; ++i) {
                if (i < NC) {
                    stage(lds + (b ^ 1) * BUFFER, i);
                    load(s + 2, i, all);
                }
                multiply(lds + b * BUFFER, i);
            }
            __syncthreads();
        }
        for (; s < count; ++s) {
            const int b = (int)s & 1;
#pragma unroll
            for (int i = 0; i < BR / 16; ++i) {
                if (i < NC && s + 1 < count) {
                    stage(lds + (b ^ 1) * BUFFER, i);
                    if (s + 2 < count) load(s + 2, i, some);
                }
                multiply(lds + b * BUFFER, i);
            }
            __syncthreads();
        }
    }
    if constexpr (SHARE > 1) {      // the waves' shares meet in LDS: a register of the tile is added up in the order of the waves (TO = TK = 1)
        float* fs = reinterpret_cast<float*>(lds);
#pragma unroll
        for (int r = 0; r < 16; ++r) fs[wave * 1024 + 64 * r + lane] = acc[0][0][r];
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            float v = fs[place * SHARE * 1024 + 64 * r + lane];
#pragma unroll
            for (int q = 1; q < SHARE; ++q) v += fs[(place * SHARE + q) * 1024 + 64 * r + lane];
            acc[0][0][r] = v;
        }
        __syncthreads();
        double* ds = reinterpret_cast<double*>(lds);
        ds[t] = bs[0];
        __syncthreads();
        double v = ds[64 * place * SHARE + lane];
#pragma unroll
        for (int q = 1; q < SHARE; ++q) v += ds[64 * (place * SHARE + q) + lane];
        bs[0] = v;
        if (wave % SHARE != 0) return;
    }
    if (TURNS > 1 && a.db && k0 < TO * WK) {
        double* ds = reinterpret_cast<double*>(lds);
#pragma unroll
        for (int i = 0; i < TO; ++i) ds[64 * (TO * wave + i) + lane] = bs[i];
        __syncthreads();
        if (turn == 0)
#pragma unroll
            for (int i = 0; i < TO; ++i)
#pragma unroll
                for (int q = 1; q < TURNS; ++q) bs[i] += ds[64 * (TO * (wave + q * SHARE) + i) + lane];
    }
    const bool last = a.splits == 1;
    auto put = [&](void* to, long at, float v) {
        if (T == LT_F32 || a.grad32) static_cast<float*>(to)[at] = v;
        else static_cast<unsigned short*>(to)[at] = (unsigned short)pack2<T == LT_F32 ? LT_F16 : T>(v, 0.0f);
    };
#pragma unroll
    for (int i = 0; i < TO; ++i)
#pragma unroll
        for (int k = 0; k < TK; ++k)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int o = o0 + 32 * (wo + i) + (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5), c = k0 + 32 * (wk + k) + (lane & 31);
                if (o < a.o && c < a.k) {
                    if (last) put(a.dw, (long)o * a.k + c, acc[i][k][r]);
                    else a.part[((long)split * a.o + o) * a.k + c] = acc[i][k][r];
                }
            }
    if (turn == 0)
#pragma unroll
        for (int i = 0; i < TO; ++i) {
            if (!sums(i)) continue;
            const double s = bs[i] + __shfl_xor(bs[i], 32);
            const int o = o0 + 32 * (wo + i) + lane;
            if (lane < 32 && o < a.o) {
                if (last) put(a.db, o, (float)s);
                else a.bias_part[(long)split * a.o + o] = s;
            }
        }
}

template <int T, int WO, int WK> __global__ __launch_bounds__(WO == 256 ? 1024 : 256, (WO == 128 && WK == 128) || (T == LT_F32 && WO != WK) ? 2 : 4) void k_dense_weights(DenseWeights a) {
    __shared__ __attribute__((aligned(16))) unsigned short lds[2 * WeightsTile<T, WO, WK>::BUFFER];
    static_assert(WeightsTile<T, WO, WK>::SHARE == 1 || sizeof(lds) >= WeightsTile<T, WO, WK>::NT / 64 * 4096, "the shares of a tile");
    dense_weights_tile<T, WO, WK>(a, blockIdx.x, lds);
}

// Both gradients of few rows in one launch: neither fills the chip, and they read the same dY.  The weight tiles, which take longer, come first.
template <int T, int WO, int WK> __global__ __launch_bounds__(256, 2) void k_dense_backward_few(DenseRows x, DenseWeights w, unsigned weight_blocks) {
    constexpr int WEIGHTS = 2 * WeightsTile<T, WO, WK>::BUFFER, ROWS = FEW_LDS * 2;
    __shared__ __attribute__((aligned(16))) unsigned short lds[WEIGHTS > ROWS ? WEIGHTS : ROWS];
    if (blockIdx.x < weight_blocks) dense_weights_tile<T, WO, WK>(w, blockIdx.x, lds);
    else dense_few<T, true>(x, blockIdx.x - weight_blocks, reinterpret_cast<float*>(lds));
}

// The pieces' sums in order, in 64 bits: a workgroup takes N of the o k + o values, G groups of threads every G-th piece each.  Many values fill the chip by themselves, few values
// of many pieces take groups (26 x 5 values of 1 024 pieces: 130 us with one thread a value, 13 with 16 groups, 6 with 64; 512 x 539 of 8: 4 us with one, 12.5 with 16;
// 384 x 384 of 56: 7 with four, 17 with one)
template <int T, int G, int N> __global__ __launch_bounds__(G * N) void k_dense_weights_sum(DenseWeights a) {
    __shared__ double sums[G > 1 ? G * N : 1];
    const int t = threadIdx.x, group = t / N;
    const long nw = (long)a.o * a.k, i = (long)blockIdx.x * N + t % N;
    const bool weight = i < nw, bias = !weight && a.db && i < nw + a.o;
    double s = 0.0;
    auto add = [&](auto* from, long stride) {      // 16 loads at a time, the last piece again beyond the end
        for (int q0 = group; q0 < a.splits; q0 += 16 * G) {
            double v[16];
#pragma unroll
            for (int u = 0; u < 16; ++u) v[u] = (double)from[min(q0 + u * G, a.splits - 1) * stride];
#pragma unroll
            for (int u = 0; u < 16; ++u) s += q0 + u * G < a.splits ? v[u] : 0.0;
        }
    };
    if (weight) add(a.part + i, nw);
    else if (bias) add(a.bias_part + (i - nw), (long)a.o);
    if constexpr (G > 1) {
        sums[t] = s;
        __syncthreads();
        if (group == 0)
#pragma unroll
            for (int q = 1; q < G; ++q) s += sums[N * q + t];
    }
    if (group != 0 || !(weight || bias)) return;
    void* to = bias ? a.db : a.dw;
    const long at = bias ? i - nw : i;
    if (T == LT_F32 || a.grad32) static_cast<float*>(to)[at] = (float)s;
    else static_cast<unsigned short*>(to)[at] = (unsigned short)pack2<T == LT_F32 ? LT_F16 : T>((float)s, 0.0f);
}

// ------------------------------------------------------------------------------------------------------------------------- checkpoints on their own
// One pass, a thread = 8 columns, HBM-bound: 786 432 x 512 bfloat16 in 250 us (1.2 GB: 4.9 TB/s, what a copy reaches), back in 225.
template <int T> __global__ __launch_bounds__(256) void k_checkpoint(const char* x, long ld, long n, int k, int is_signed, uint8_t* codes, uint8_t* scales) {
    const int cpr = ((k + 31) >> 5) * 4;      // 8-column chunks a row; a block's four lie in four neighbouring lanes
    const long total = n * cpr;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < ((total + 63) & ~63L); i += (long)gridDim.x * 256) {      // whole waves: encode8 exchanges between lanes
        const bool in = i < total;
        const long p = in ? i / cpr : 0;
        const int c = 8 * (int)(in ? i - p * cpr : 0);
        u32x2 q; unsigned s;
        encode8<T>(in ? load8<T>(x + p * ld * Bytes<T>::v, c, k) : zero8<T>(), is_signed != 0, q, s);
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
        const u32x2 codes = *reinterpret_cast<const u32x2*>(a.codes + 8 * i);
        const unsigned scale = a.scales[i >> 2];
        if (large_block<T>(scale)) decode8_large<T>(codes, scale, a.is_signed != 0, f);
        else decode8(codes, scale, a.is_signed != 0, f);
        store8<T>(out + p * ld * Bytes<T>::v, c, k, from_floats<T>(f));
    }
}

// Few rows: 1 024 workgroups of k_dense_few or less, four a compute unit.  (us, k_dense_few / the others, at 1 024 rows of 512 -> 512: float32 14 / 35, bfloat16 8 / 16; 2 048: 22 / 36 and
// 13 / 16; 4 096: 39 / 37 and 21 / 17; 20 000 of 512 -> 4 bfloat16: 8 / 13)
long few_blocks(long n, int o) { return ((n + 31) / 32) * ((o + 31) / 32); }
constexpr long FEW_BLOCKS = 1024;

// Which form Y = act(A B + bias) runs in, and the fragments' memory.  For the 16-bit types, beyond few rows: the narrow form for at most 32 outputs (100 000 rows of 26 -> 18: 8 us, 30
// in the tall form; of 500 -> 32: 34, 55; its weights leave room for four workgroups on a compute unit up to 352 columns and for three up to 512: 262 144 rows of 512 -> 32 66 us,
// of 528 in the tall form 112), else the tall form once its tiles of 128 rows give every compute unit one (32 767 rows of 512 -> 512 in k_dense_rows 36 us, 32 768 here 30; rows of 8
// elements at least: it reads whole chunks; up to 8 passes, whose biases lie in LDS beside the two buffers).  A pass makes 256 outputs.  (Beyond 6 passes the biases, for which the input
// gradient keeps room too, leave a compute unit one workgroup: 65 536 x 512 bfloat16 -> 1 536 157 us, 1 537 229, 2 048 254, 2 049 in k_dense_rows 261.)
struct RowsPlan { bool few, narrow, tall; int passes, steps; };
RowsPlan rows_plan(int type, long n, int r, int o) {
    RowsPlan p{};
    p.passes = (o + 255) / 256;
    p.few = few_blocks(n, o) <= FEW_BLOCKS;
    p.narrow = !p.few && type != LT_F32 && o <= 32 && r <= 512;
    p.tall = !p.few && !p.narrow && type != LT_F32 && n >= 256 * TALL_ROWS && r >= 8 && p.passes <= 8;
    p.steps = (r + 63) / 64 * 4;
    return p;
}

template <int T, int MODE, int COLS> hipError_t dense_tall(const DenseRows& a, const RowsPlan& p, u32x4* wf, hipStream_t s) {
    const int tiles = p.passes * 8;
    const size_t bytes = 4 * (size_t)TALL_ROWS * COLS + 4 * 2560 + p.passes * 256 * 4;
    // (once for each device and kernel: more LDS than the default 64 KB)
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    static std::atomic<unsigned long long> set{0};
    if (dev > 63 || !(set.load(std::memory_order_acquire) >> dev & 1)) {
        e = hipFuncSetAttribute(reinterpret_cast<const void*>(&k_dense_tall<T, MODE, COLS>), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
        if (e != hipSuccess) return e;
        if (dev <= 63) set.fetch_or(1ull << dev, std::memory_order_release);
    }
    hipLaunchKernelGGL((k_dense_fragments<T, MODE == TALL_DX>), dim3((unsigned)(tiles * (p.steps / 4))), dim3(256), 0, s, a, wf, tiles, p.steps);
    hipLaunchKernelGGL((k_dense_tall<T, MODE, COLS>), dim3(512), dim3(256), bytes, s, a, wf, p.passes);
    return hipGetLastError();
}
template <int T, int MODE> hipError_t dense_tall(const DenseRows& a, const RowsPlan& p, u32x4* wf, hipStream_t s) {
    return a.r <= 64 ? dense_tall<T, MODE, 64>(a, p, wf, s) : dense_tall<T, MODE, 128>(a, p, wf, s);
}

template <int T, bool DX> hipError_t dense_rows(const DenseRows& a, void* ws, hipStream_t s) {
    const RowsPlan p = rows_plan(T, a.n, a.r, a.o);
    if constexpr (T != LT_F32) {
        if (p.narrow) {
            const long groups = (a.n + 127) / 128;
            hipLaunchKernelGGL((k_dense_narrow<T, DX>), dim3((unsigned)(groups < 2048 ? groups : 2048)), dim3(256), (FEW_LDS + 256 * ((a.r + 15) / 16)) * sizeof(float), s, a);
            return hipGetLastError();
        }
        if (p.tall) {
            u32x4* wf = static_cast<u32x4*>(ws);
            if constexpr (DX) return dense_tall<T, TALL_DX>(a, p, wf, s);
            else return !a.codes ? dense_tall<T, TALL_Y>(a, p, wf, s) : a.relu ? dense_tall<T, TALL_RELU_KEEP>(a, p, wf, s) : dense_tall<T, TALL_KEEP>(a, p, wf, s);
        }
    }
    if (p.few) {
        hipLaunchKernelGGL((k_dense_few<T, DX>), dim3((unsigned)few_blocks(a.n, a.o)), dim3(256), 0, s, a);
        return hipGetLastError();
    }
    const long pt = ((a.n + 127) / 128 + 7) / 8 * 8;
    // half as wide where 128 would compute much beyond the layer (float32, us: 512 -> 4 85 instead of 131, 96 -> 20 29 instead of 52, 561 -> 161 389 instead of 433; 512 -> 540 248
    // instead of 241)
    if (a.o <= 192 && (a.o - 1) % 128 < 64) hipLaunchKernelGGL((k_dense_rows<T, DX, 128, 64>), dim3((unsigned)(pt * ((a.o + 63) / 64))), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_dense_rows<T, DX, 128, 128>), dim3((unsigned)(pt * ((a.o + 127) / 128))), dim3(256), 0, s, a);
    return hipGetLastError();
}

// The weight gradient's tile and how many pieces the rows are cut into (functions of the sizes alone)
struct WeightsPlan { int wo, wk, tiles, splits; };
WeightsPlan weights_plan(int type, long n, int k, int o) {
    WeightsPlan p;
    const long t4 = (long)((k + 127) / 128) * ((o + 127) / 128), t8 = (long)((k + 255) / 256) * ((o + 255) / 256);
    const long steps = type == LT_F32 ? (n + 31) / 32 : (n + 63) / 64;
    // 256 x 256 where that computes at most half as much again beyond the layer's edges and each of the 256 compute units has some steps to do; pieces of two steps at least
    // (1 003 x 539 -> 512: 18 us; 25 in 256-wide tiles, 24 in pieces of one step).  A side of at most 32 columns takes 32-wide tiles (512 -> 4 float32: 9 us instead of 12 for 2 048
    // rows, 15 instead of 18 for 16 384; 26 <- 5 bfloat16: 15 instead of 100 for 730 935)
    p.wo = p.wk = 2 * 4 * t8 <= 3 * t4 && steps * t8 >= 4 * 256 ? 256 : 128;
    if (p.wo == 128) {
        if (o <= 32) p.wo = 32;
        if (k <= 32) p.wk = 32;
    }
    p.tiles = (int)(((long)(k + p.wk - 1) / p.wk) * ((o + p.wo - 1) / p.wo));
    long s = (p.wo == 256 ? 256 : p.wo == 128 && p.wk == 128 ? 512 : 1024) / p.tiles;      // one workgroup a compute unit, two, four
    if (s > steps / 2) s = steps / 2;
    p.splits = (int)(s < 1 ? 1 : s);
    return p;
}

// (x: the input gradient where that is asked for too and runs in the few-rows form, or null)
template <int T, int WO, int WK> void dense_weights(const DenseWeights& a, unsigned blocks, const DenseRows* x, hipStream_t s) {
    if (x) hipLaunchKernelGGL((k_dense_backward_few<T, WO, WK>), dim3(blocks + (unsigned)few_blocks(x->n, x->o)), dim3(256), 0, s, *x, a, blocks);
    else hipLaunchKernelGGL((k_dense_weights<T, WO, WK>), dim3(blocks), dim3(256), 0, s, a);
}
template <int T> hipError_t dense_weights(const DenseWeights& a, const DenseRows* x, hipStream_t s) {
    const WeightsPlan p = weights_plan(T, a.n, a.k, a.o);
    const unsigned blocks = (unsigned)((p.splits + 7) / 8 * 8 * p.tiles);
    if (p.wo == 256) {
        if (x) hipLaunchKernelGGL((k_dense_few<T, true>), dim3((unsigned)few_blocks(x->n, x->o)), dim3(256), 0, s, *x);
        hipLaunchKernelGGL((k_dense_weights<T, 256, 256>), dim3(blocks), dim3(1024), 0, s, a);
    } else if (p.wo == 32 && p.wk == 32) dense_weights<T, 32, 32>(a, blocks, x, s);
    else if (p.wo == 32) dense_weights<T, 32, 128>(a, blocks, x, s);
    else if (p.wk == 32) dense_weights<T, 128, 32>(a, blocks, x, s);
    else dense_weights<T, 128, 128>(a, blocks, x, s);
    if (a.splits > 1) {
        const long m = (long)a.o * a.k + a.o;
        if (a.splits <= 16) hipLaunchKernelGGL((k_dense_weights_sum<T, 1, 256>), dim3((unsigned)((m + 255) / 256)), dim3(256), 0, s, a);
        else if (m >= 16384) hipLaunchKernelGGL((k_dense_weights_sum<T, 4, 64>), dim3((unsigned)((m + 63) / 64)), dim3(256), 0, s, a);
        else if (a.splits <= 256) hipLaunchKernelGGL((k_dense_weights_sum<T, 16, 64>), dim3((unsigned)((m + 63) / 64)), dim3(1024), 0, s, a);
        else hipLaunchKernelGGL((k_dense_weights_sum<T, 64, 16>), dim3((unsigned)((m + 15) / 16)), dim3(1024), 0, s, a);
    }
    return hipGetLastError();
}

unsigned chunk_grid(long n, int k) {
    const long blocks = (n * (((k + 31) >> 5) * 4) + 255) / 256;
    return (unsigned)(blocks < 16384 ? blocks : 16384);
}

}  // namespace

int dense_weight_splits(int type, long n, int k, int o) { return weights_plan(type, n, k, o).splits; }

size_t dense_rows_bytes(int type, long n, int r, int o) {
    const RowsPlan p = rows_plan(type, n, r, o);
    return p.tall ? (size_t)p.passes * 8 * p.steps * 1024 : 0;
}

hipError_t launch_dense_rows(int type, bool input_gradient, const DenseRows& a, void* ws, hipStream_t s) {
    if (input_gradient) return type == LT_F32 ? dense_rows<LT_F32, true>(a, ws, s) : type == LT_BF16 ? dense_rows<LT_BF16, true>(a, ws, s) : dense_rows<LT_F16, true>(a, ws, s);
    return type == LT_F32 ? dense_rows<LT_F32, false>(a, ws, s) : type == LT_BF16 ? dense_rows<LT_BF16, false>(a, ws, s) : dense_rows<LT_F16, false>(a, ws, s);
}

hipError_t launch_dense_backward(int type, const DenseRows* x, const DenseWeights* w, void* ws, hipStream_t s) {
    const bool together = x && w && x->n > 0 && rows_plan(type, x->n, x->r, x->o).few;
    if (x && x->n > 0 && !together) {
        const hipError_t e = launch_dense_rows(type, true, *x, ws, s);
        if (e != hipSuccess) return e;
    }
    if (!w) return hipSuccess;
    const DenseRows* both = together ? x : nullptr;
    return type == LT_F32 ? dense_weights<LT_F32>(*w, both, s) : type == LT_BF16 ? dense_weights<LT_BF16>(*w, both, s) : dense_weights<LT_F16>(*w, both, s);
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
