// Table rows by index with a scale (a code for the view of each ray), and the table's gradient by sorted tokens.
//
//   out[p][c] = scale * table[index[p / per]][c]            d table[t][c] = scale * sum over the rows p with index[p / per] = t of dOut[p][c]
//
// A negative index is a row without a code: zeros, no gradient.  An index beyond the table reads NaN (a wrong index shows) and has no gradient.
//
// The gradient is bound by reading dOut once, in an order that the tokens set.  Up to 16 384 positions one launch does it all (k_lookup_few).  Otherwise the positions are sorted
// by token (stable, so a token's rows keep their order), the sorted rows are cut into pieces of equal length — a token that most rows share (a batch drawn from few views)
// costs no more than any other — and each piece adds up its runs of equal tokens in 32 bits.  A run inside one piece is finished there; the pieces of a longer run are
// joined in order by k_lookup_join.  No atomics on values: the same inputs give the same bits.
//
// Measured: lookup 786 432 x 32 bfloat16 12.5 us (50 MB: 4.0 TB/s).  Gradient of 4 096 positions, 200 x 48: 6.4 us.  Of 640 000, 65 536 x 64 float32: 81 to 94 us — each of two
// sorting passes 6.7 (counts) + 3.7 (their sums) + 11 (scatter), rows 31 (164 MB: 5.3 TB/s), joins 11.
#include "layer_elems.h"
#include "layers.h"

namespace ibl {

namespace {

constexpr int SMALL = 4096;          // positions that one workgroup sorts in LDS
constexpr int TILE = 2048;           // positions a workgroup of the large sort takes
constexpr int BINS = 512;            // at most 9 bits a pass
typedef u32x2 Entry;                 // a sorted position: its key, itself (one store where the sort scatters)

__device__ __forceinline__ long index_at(const void* index, int index64, long i) {
    return index64 ? static_cast<const long long*>(index)[i] : (long)static_cast<const int*>(index)[i];
}
// a position's sort key: its token, or v (behind all tokens) where it has none
__device__ __forceinline__ unsigned key_at(const LookupGrad& a, long i) {
    const long t = index_at(a.index, a.index64, i);
    return t >= 0 && t < a.v ? (unsigned)t : (unsigned)a.v;
}

// thread `t` of `threads` clears its share of a table of 2- or 4-byte elements
__device__ __forceinline__ void clear(void* table, size_t bytes, size_t t, size_t threads) {
    size_t whole = 0;
    if ((reinterpret_cast<uintptr_t>(table) & 15) == 0) {
        whole = bytes / 16;
        for (size_t i = t; i < whole; i += threads) static_cast<u32x4*>(table)[i] = u32x4{0, 0, 0, 0};
    }
    for (size_t i = 8 * whole + t; i < bytes / 2; i += threads) static_cast<unsigned short*>(table)[i] = 0;
}

template <int T> __global__ __launch_bounds__(256) void k_lookup(Lookup a) {
    const int cpr = (a.d + 7) >> 3;
    const long total = a.n * a.per * cpr;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
        const long row = i / cpr;
        const int c = 8 * (int)(i - row * cpr);
        const long t = index_at(a.index, a.index64, a.per == 1 ? row : row / a.per);
        float f[8];
        if (t >= 0 && t < a.v) {
            to_floats<T>(load8<T>(static_cast<const char*>(a.table) + t * a.ld_table * Bytes<T>::v, c, a.d), f);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] *= a.scale;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = t < 0 ? 0.0f : __builtin_nanf("");
        }
        store8<T>(static_cast<char*>(a.out) + row * a.ld_out * Bytes<T>::v, c, a.d, from_floats<T>(f));
    }
}

// ------------------------------------------------------------------------------------------------------------------------------------------------ sorting
// Lanes of the wave whose digit equals this lane's (only lanes with `in` count)
__device__ __forceinline__ unsigned long long peers(unsigned digit, bool in) {
    unsigned long long m = __ballot(in);
#pragma unroll
    for (int b = 0; b < 9; ++b) {      // (a shorter digit's upper bits are equal in all lanes)
        const bool one = (digit >> b) & 1;
        const unsigned long long v = __ballot(one);
        m &= one ? v : ~v;
    }
    return m;
}

// One stable pass over `rounds` x 64 keys of each wave: the key's rank among the wave's keys of the same digit, the wave's digit counts in hist[wave][BINS]
template <int WAVES> __device__ __forceinline__ unsigned rank_in_wave(unsigned digit, bool in, unsigned* hist, int wave, int lane) {
    const unsigned long long m = peers(digit, in);
    unsigned before = 0;
    if (in) before = hist[wave * BINS + digit];
    const unsigned lower = __popcll(m & ((1ull << lane) - 1));
    __builtin_amdgcn_wave_barrier();
    if (in && lower == 0) hist[wave * BINS + digit] = before + (unsigned)__popcll(m);
    __builtin_amdgcn_wave_barrier();
    return before + lower;
}

// up to SMALL positions, all passes in one workgroup of 16 waves; wave w holds positions 256 w .. 256 w + 255
__global__ __launch_bounds__(1024) void k_sort_small(LookupGrad a, int passes, int bits, Entry* sorted, size_t zero_bytes) {
    __shared__ unsigned lk[SMALL], lp[SMALL];
    __shared__ unsigned hist[16 * BINS];
    __shared__ unsigned base[BINS];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, n = (int)a.n;
    clear(a.dtable, zero_bytes, t, 1024);
    for (int i = t; i < n; i += 1024) { lk[i] = key_at(a, i); lp[i] = (unsigned)i; }
    __syncthreads();
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = pass * bits;
        const unsigned mask = (1u << bits) - 1;
        for (int i = t; i < 16 * BINS; i += 1024) hist[i] = 0;
        __syncthreads();
        unsigned k[4], p[4], r[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int i = 256 * wave + 64 * q + lane;
            const bool in = i < n;
            k[q] = in ? lk[i] : 0;
            p[q] = in ? lp[i] : 0;
            r[q] = rank_in_wave<16>((k[q] >> shift) & mask, in, hist, wave, lane);
        }
        __syncthreads();
        // the waves' counts of a digit become exclusive sums; base = the digit's total
        if (t < BINS) {
            unsigned s = 0;
#pragma unroll
            for (int w = 0; w < 16; ++w) { const unsigned h = hist[w * BINS + t]; hist[w * BINS + t] = s; s += h; }
            base[t] = s;
        }
        __syncthreads();
        if (t < 64) {      // exclusive sums over the digits, 8 a lane
            unsigned v[BINS / 64], s = 0;
#pragma unroll
            for (int q = 0; q < BINS / 64; ++q) { v[q] = base[t * (BINS / 64) + q]; s += v[q]; }
            unsigned x = s;
#pragma unroll
            for (int m = 1; m < 64; m <<= 1) { const unsigned y = __shfl_up(x, m); if (lane >= m) x += y; }
            x -= s;
#pragma unroll
            for (int q = 0; q < BINS / 64; ++q) { base[t * (BINS / 64) + q] = x; x += v[q]; }
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int i = 256 * wave + 64 * q + lane;
            if (i < n) {
                const unsigned dg = (k[q] >> shift) & mask, at = base[dg] + hist[wave * BINS + dg] + r[q];
                lk[at] = k[q];
                lp[at] = p[q];
            }
        }
        __syncthreads();
    }
    for (int i = t; i < n; i += 1024) sorted[i] = Entry{lk[i], lp[i]};
}

template <class Key> __device__ __forceinline__ void count_tile(Key key, long n, int shift, int bits, unsigned* hist) {
    const long i0 = (long)blockIdx.x * TILE + threadIdx.x;
    unsigned k[TILE / 256];
#pragma unroll
    for (int q = 0; q < TILE / 256; ++q) k[q] = key(min(i0 + 256 * q, n - 1));
#pragma unroll
    for (int q = 0; q < TILE / 256; ++q)
        if (i0 + 256 * q < n) atomicAdd(&hist[(k[q] >> shift) & ((1u << bits) - 1)], 1u);
}

// Large sort, one pass = three launches: digit counts of each tile, their exclusive sums along the tiles (one workgroup a digit), the scatter.
// The first pass reads the caller's index; its counting launch also clears the gradient table (tokens that no row has keep zero).
__global__ __launch_bounds__(256) void k_sort_count(LookupGrad a, const Entry* from, int shift, int bits, unsigned* counts, size_t zero_bytes) {
    __shared__ unsigned hist[BINS];
    for (int i = threadIdx.x; i < BINS; i += 256) hist[i] = 0;
    __syncthreads();
    if (from) count_tile([&](long i) { return from[i][0]; }, a.n, shift, bits, hist);
    else count_tile([&](long i) { return key_at(a, i); }, a.n, shift, bits, hist);
    __syncthreads();
    for (int i = threadIdx.x; i < (1 << bits); i += 256) counts[(size_t)i * gridDim.x + blockIdx.x] = hist[i];
    clear(a.dtable, zero_bytes, (size_t)blockIdx.x * 256 + threadIdx.x, (size_t)gridDim.x * 256);
}

__global__ __launch_bounds__(256) void k_sort_scan(unsigned* counts, int tiles, unsigned* totals) {
    __shared__ unsigned part[4];
    unsigned* row = counts + (size_t)blockIdx.x * tiles;
    const int t = threadIdx.x, lane = t & 63;
    unsigned carry = 0;
    for (int i0 = 0; i0 < tiles; i0 += 256) {
        const unsigned v = i0 + t < tiles ? row[i0 + t] : 0;
        unsigned x = v;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) { const unsigned y = __shfl_up(x, m); if (lane >= m) x += y; }
        if (lane == 63) part[t >> 6] = x;
        __syncthreads();
        unsigned before = carry, all = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) { if (w < (t >> 6)) before += part[w]; all += part[w]; }
        if (i0 + t < tiles) row[i0 + t] = before + x - v;
        carry += all;
        __syncthreads();
    }
    if (t == 0) totals[blockIdx.x] = carry;
}

__global__ __launch_bounds__(256) void k_sort_scatter(LookupGrad a, const Entry* from, int shift, int bits, const unsigned* counts, const unsigned* totals, Entry* to) {
    __shared__ unsigned hist[4 * BINS];
    __shared__ unsigned base[BINS];
    constexpr int Q = TILE / 256, B = BINS / 256;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, bins = 1 << bits;
    const long i0 = (long)blockIdx.x * TILE + (long)wave * (TILE / 4);
    // everything the tile needs is asked for at once: its keys and positions, its counts, the digits' totals
    unsigned k[Q], p[Q], r[Q], before[B], total[B];
    if (from) {
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            const Entry e = from[min(i0 + 64 * q + lane, a.n - 1)];
            k[q] = e[0];
            p[q] = e[1];
        }
    } else {
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            const long i = min(i0 + 64 * q + lane, a.n - 1);
            k[q] = key_at(a, i);
            p[q] = (unsigned)i;
        }
    }
#pragma unroll
    for (int q = 0; q < B; ++q) {
        const int d = min(t + 256 * q, bins - 1);
        before[q] = counts[(size_t)d * gridDim.x + blockIdx.x];
        total[q] = totals[d];
    }
    for (int i = t; i < 4 * BINS; i += 256) hist[i] = 0;
#pragma unroll
    for (int q = 0; q < B; ++q) base[t + 256 * q] = t + 256 * q < bins ? total[q] : 0;
    __syncthreads();
    if (t < 64) {
        unsigned v[BINS / 64], s = 0;
#pragma unroll
        for (int q = 0; q < BINS / 64; ++q) { v[q] = base[t * (BINS / 64) + q]; s += v[q]; }
        unsigned x = s;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) { const unsigned y = __shfl_up(x, m); if (lane >= m) x += y; }
        x -= s;
#pragma unroll
        for (int q = 0; q < BINS / 64; ++q) { base[t * (BINS / 64) + q] = x; x += v[q]; }
    }
#pragma unroll
    for (int q = 0; q < Q; ++q) r[q] = rank_in_wave<4>((k[q] >> shift) & (bins - 1), i0 + 64 * q + lane < a.n, hist, wave, lane);
    __syncthreads();
#pragma unroll
    for (int q = 0; q < B; ++q) {
        const int i = t + 256 * q;
        if (i < bins) {
            unsigned s = base[i] + before[q];
#pragma unroll
            for (int w = 0; w < 4; ++w) { const unsigned h = hist[w * BINS + i]; hist[w * BINS + i] = s; s += h; }
        }
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < Q; ++q)
        if (i0 + 64 * q + lane < a.n) {
            const unsigned at = hist[wave * BINS + ((k[q] >> shift) & (bins - 1))] + r[q];
            to[at] = Entry{k[q], p[q]};
        }
}

// ------------------------------------------------------------------------------------------------------------------------------------------------ summing
template <int T> __device__ __forceinline__ void put_sum(const LookupGrad& a, unsigned token, int c, const float (&s)[8]) {
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = s[e] * a.scale;
    store8<T>(static_cast<char*>(a.dtable) + (size_t)token * a.d * Bytes<T>::v, c, a.d, from_floats<T>(f));
}

// Where a thread's 8 columns begin: in rows of 8 and more the last chunk moves back to end with the row, so that every chunk is whole — two neighbours then hold some columns'
// sums twice, the same bits — and loads need no branch.  WIDE: such rows.
template <bool WIDE> __device__ __forceinline__ int chunk_at(int chunk, int d) { return WIDE ? min(8 * chunk, d - 8) : 8 * chunk; }
template <int T, bool WIDE> __device__ __forceinline__ Raw8<T> load_chunk(const char* row, int c, int d) {
    if constexpr (WIDE) return load8_whole<T>(row, c);
    else return load8<T>(row, c, d);
}

// A thread = 8 columns of one piece: sorted rows [piece * len, piece * len + len), sorted row i = row i % per of the entry i / per.  part [pieces][2][8 cpr]: the sum of the
// run that comes in from the piece before (0) and of the run that goes on into the next (1).
template <int T, bool WIDE> __global__ __launch_bounds__(256) void k_lookup_sum(LookupGrad a, const Entry* sorted, long pieces, int len, float* part) {
    constexpr int U = 8;      // rows in flight
    const int cpr = (a.d + 7) >> 3;
    const long id = (long)blockIdx.x * 256 + threadIdx.x;
    const long piece = id / cpr;
    if (piece >= pieces) return;
    const int c = chunk_at<WIDE>((int)(id - piece * cpr), a.d);
    const long rows = a.n * a.per, i0 = piece * len, i1 = i0 + len < rows ? i0 + len : rows;
    const unsigned none = (unsigned)a.v;
    float* out = part + (size_t)piece * 2 * 8 * cpr + c;
    auto keep = [&](int which, const float (&s)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) out[which * 8 * cpr + e] = s[e];
    };
    unsigned cur = sorted[i0 / a.per][0];
    bool coming = i0 > 0 && sorted[(i0 - 1) / a.per][0] == cur;
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (long i = i0; i < i1; i += U) {
        unsigned k[U];
        long at[U];
        Raw8<T> v[U];
        long e = i / a.per, q = i - e * a.per;
#pragma unroll
        for (int u = 0; u < U; ++u) {      // (rows beyond the piece: its last again)
            const Entry x = sorted[e];
            k[u] = x[0];
            at[u] = (long)x[1] * a.per + q;
            if (i + u + 1 < i1 && ++q == a.per) { q = 0; ++e; }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = load_chunk<T, WIDE>(static_cast<const char*>(a.dout) + at[u] * a.ld_dout * Bytes<T>::v, c, a.d);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i + u >= i1) break;
            if (k[u] != cur) {
                if (coming) keep(0, s);
                else if (cur != none) put_sum<T>(a, cur, c, s);
                coming = false;
                cur = k[u];
#pragma unroll
                for (int x = 0; x < 8; ++x) s[x] = 0.0f;
            }
            float f[8];
            to_floats<T>(v[u], f);
#pragma unroll
            for (int x = 0; x < 8; ++x) s[x] += f[x];
        }
    }
    if (cur == none) return;
    if (coming) keep(0, s);
    else if (i1 < rows && sorted[i1 / a.per][0] == cur) keep(1, s);
    else put_sum<T>(a, cur, c, s);
}

// Runs that begin in a piece and go on: the run's partial sums — its own and those of the pieces it comes into — are added up.  A wave looks at one piece; a short run (the usual
// case: it ends in the next piece) is its own work, lane by column; a long one is done by the workgroup: each thread a column and every G-th piece, then the G sums in order.
template <int T> __device__ __forceinline__ void put_one(const LookupGrad& a, unsigned token, int c, float s) {
    const size_t at = (size_t)token * a.d + c;
    s *= a.scale;
    if constexpr (T == LT_F32) static_cast<float*>(a.dtable)[at] = s;
    else static_cast<unsigned short*>(a.dtable)[at] = (unsigned short)pack2<T>(s, 0.0f);
}
template <int T> __global__ __launch_bounds__(256) void k_lookup_join(LookupGrad a, const Entry* sorted, long pieces, int len, const float* part) {
    constexpr long SHORT = 16;
    __shared__ f32x4 sums[256];
    __shared__ unsigned token[4];
    __shared__ int goes_on[4];      // pieces that the run comes into, where it is a long one
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), w = 8 * ((a.d + 7) >> 3);
    const long rows = a.n * a.per, piece = (long)blockIdx.x * 4 + wave, i0 = piece * len, i1 = i0 + len;
    long more = 0;
    unsigned tok = 0;
    if (i1 < rows) {
        tok = sorted[(i1 - 1) / a.per][0];
        if (tok != (unsigned)a.v && sorted[i1 / a.per][0] == tok && !(i0 > 0 && sorted[(i0 - 1) / a.per][0] == tok)) {      // (else: no run goes on, or it began in an earlier piece)
            more = 1;
            if (i1 + len < rows && sorted[(i1 + len) / a.per][0] == tok) {      // further than the next piece: where the run ends
                long lo = (i1 + len) / a.per, hi = a.n;
                while (lo < hi) {
                    const long m = (lo + hi) >> 1;
                    if (sorted[m][0] <= tok) lo = m + 1; else hi = m;
                }
                more = (lo * a.per - 1) / len - piece;
            }
        }
    }
    const float* first = part + (size_t)piece * 2 * w;
    if (more > 0 && more <= SHORT)
        for (int c = lane; c < a.d; c += 64) {
            float s = first[w + c];
            for (long q = 0; q < more; ++q) s += first[(size_t)(q + 1) * 2 * w + c];
            put_one<T>(a, tok, c, s);
        }
    if (lane == 0) { token[wave] = tok; goes_on[wave] = more > SHORT ? (int)more : 0; }
    __syncthreads();
    for (int y = 0; y < 4; ++y) {
        const int n = goes_on[y];
        if (n == 0) continue;
        const float* from = part + (size_t)((long)blockIdx.x * 4 + y) * 2 * w;
        const int quads = w >> 2;
        for (int q0 = 0; q0 < quads; q0 += 256) {
            const int cols = quads - q0 < 256 ? quads - q0 : 256, g = 256 / cols, c = t % cols, z = t / cols;
            f32x4 s = {0.f, 0.f, 0.f, 0.f};
            if (z < g) {
                if (z == 0) s = *reinterpret_cast<const f32x4*>(from + w + 4 * (q0 + c));
                const float* p = from + 2 * w + 4 * (q0 + c);
#pragma unroll 8
                for (int q = z; q < n; q += g) s += *reinterpret_cast<const f32x4*>(p + (size_t)q * 2 * w);
            }
            sums[t] = s;
            __syncthreads();
            if (t < cols) {
                f32x4 r = sums[t];
                for (int q = 1; q < g; ++q) r += sums[q * cols + t];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (4 * (q0 + t) + e < a.d) put_one<T>(a, token[y], 4 * (q0 + t) + e, r[e]);
            }
            __syncthreads();
        }
    }
}

// Few positions, no sort: a workgroup takes every 2^bits-th token (neighbours tend to be read alike, and go to different workgroups), reads every key and keeps the positions of its
// tokens, in order; one launch writes the whole table, zeros too.  (The worst tokens are those alike in their low bits, a column of a grid of 256 cells a row: one workgroup has all
// of them.  4 096 positions on multiples of 256 take 670 us, 16 384 2.6 ms; anywhere 13 and 31, on neighbours 10 and 16.)  One token is summed by the whole workgroup, and so is a token of several with many rows; the other
// tokens are a wave's work each (where positions are fewer than tokens, found by their first position).
constexpr int MANY = 256;      // rows
constexpr int FEW = 16384;     // positions
// rows, elements of dOut, elements a token on the average: beyond these one workgroup may have too much to read alone (8 192 rows of one token x 256 float32: 87 us, 27 in pieces;
// 13 030 positions of 2 495 x 1: 19, 43 in pieces)
constexpr long FEW_ROWS = 65536, FEW_ELEMENTS = 1 << 21, FEW_SHARE = 32768;
struct FewLds {
    unsigned short pos[FEW], tok[FEW];
    unsigned short mine[16][64];
    unsigned many[FEW_ROWS / MANY];
    int wave[16], n_many;
    float sums[1024 * 8];
};
// the positions of the tokens t0, t0 + 2^bits, t0 + 2 * 2^bits, ... (t0 alone: bits = 32), in order
__device__ __forceinline__ int few_collect(const LookupGrad& a, unsigned t0, int bits, FewLds& l) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, n = (int)a.n;
    auto ask = [&](int i0, unsigned (&k)[4]) {
#pragma unroll
        for (int q = 0; q < 4; ++q) k[q] = key_at(a, min(i0 + 256 * wave + 64 * q + lane, n - 1));
    };
    unsigned next[4];
    ask(0, next);
    int total = 0;
    for (int i0 = 0; i0 < n; i0 += 4096) {      // 256 positions a wave
        unsigned k[4];
        int at[4], count = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) k[q] = next[q];
        if (i0 + 4096 < n) ask(i0 + 4096, next);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const bool in = i0 + 256 * wave + 64 * q + lane < n && (bits < 32 ? (k[q] & ((1u << bits) - 1)) == t0 : k[q] == t0) && k[q] < (unsigned)a.v;
            const unsigned long long m = __ballot(in);
            at[q] = in ? count + __popcll(m & ((1ull << lane) - 1)) : -1;
            count += __popcll(m);
        }
        if (lane == 0) l.wave[wave] = count;
        __syncthreads();
        int before = total;
#pragma unroll
        for (int w = 0; w < 16; ++w) { if (w < wave) before += l.wave[w]; total += l.wave[w]; }
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (at[q] >= 0) {
                l.pos[before + at[q]] = (unsigned short)(i0 + 256 * wave + 64 * q + lane);
                l.tok[before + at[q]] = (unsigned short)(bits < 32 ? k[q] >> bits : 0);
            }
        __syncthreads();
    }
    return total;
}
// rows first, first + step, ... below `rows` of the positions in `pos`, 8 columns from c on
template <int T, bool WIDE> __device__ __forceinline__ void few_rows(const LookupGrad& a, const unsigned short* pos, int rows, int first, int step, int c, float (&s)[8]) {
    constexpr int U = 8;
    const int per = (int)a.per;
    for (int i0 = first; i0 < rows; i0 += U * step) {
        Raw8<T> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = min(i0 + u * step, rows - 1), e = i / per;
            v[u] = load_chunk<T, WIDE>(static_cast<const char*>(a.dout) + ((long)pos[e] * per + (i - e * per)) * a.ld_dout * Bytes<T>::v, c, a.d);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + u * step < rows) {
                float f[8];
                to_floats<T>(v[u], f);
#pragma unroll
                for (int x = 0; x < 8; ++x) s[x] += f[x];
            }
    }
}
// one token, all its `m` positions in the list: thread = 8 columns of every g-th row; the g sums meet in two steps
template <int T, bool WIDE> __device__ __forceinline__ void few_whole(const LookupGrad& a, unsigned token, int m, FewLds& l) {
    const int t = threadIdx.x, cpr = (a.d + 7) >> 3, rows = m * (int)a.per;
    for (int c0 = 0; c0 < cpr; c0 += 128) {
        const int chunks = min(cpr - c0, 128), cols = 8 * chunks, g = min(1024 / chunks, max(rows, 1)), parts = min(min(1024 / cols, 32), g), y = t / chunks, c = chunk_at<WIDE>(c0 + t % chunks, a.d);
        float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (y < g) {
            few_rows<T, WIDE>(a, l.pos, rows, y, g, c, s);
#pragma unroll
            for (int x = 0; x < 8; ++x)
                if (c + x >= 8 * c0) l.sums[y * cols + c - 8 * c0 + x] = s[x];
        }
        __syncthreads();
        const int part = t / cols, col = t % cols;
        float r = 0.0f;
        if (part < parts)
            for (int q = part; q < g; q += parts) r += l.sums[q * cols + col];
        __syncthreads();
        l.sums[t] = r;
        __syncthreads();
        if (t < cols && 8 * c0 + t < a.d) {
            for (int q = 1; q < parts; ++q) r += l.sums[q * cols + t];
            put_one<T>(a, token, 8 * c0 + t, r);
        }
        __syncthreads();
    }
}
template <int T, bool WIDE> __global__ __launch_bounds__(1024) void k_lookup_few(LookupGrad a, int bits) {
    __shared__ FewLds l;
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), cpr = (a.d + 7) >> 3, per = (int)a.per;
    const unsigned t0 = blockIdx.x;
    if (t == 0) l.n_many = 0;
    const int m = few_collect(a, t0, bits, l);
    if (bits == 32) {
        few_whole<T, WIDE>(a, t0, m, l);
        return;
    }
    const int tokens = (int)(((unsigned)a.v - t0 + (1u << bits) - 1) >> bits);
    for (int i = t; i < tokens * cpr; i += 1024) {
        const int x = i / cpr;
        store8<T>(static_cast<char*>(a.dtable) + (size_t)(t0 + ((unsigned)x << bits)) * a.d * Bytes<T>::v, 8 * (i - x * cpr), a.d, zero8<T>());
    }
    __syncthreads();
    float* sums = l.sums + 512 * wave;
    const bool by_token = m >= tokens;      // (else by position, at a token's first)
    for (int x = wave; x < (by_token ? tokens : m); x += 16) {
        const unsigned tl = by_token ? (unsigned)x : (unsigned)__builtin_amdgcn_readfirstlane((int)l.tok[x]);
        const int first = by_token ? 0 : x;
        int count = 0;
        bool earlier = false;
        for (int j = 0; j < m && !earlier; j += 64) {
            const unsigned long long mask = __ballot(j + lane < m && l.tok[min(j + lane, m - 1)] == tl);
            earlier = mask != 0 && count == 0 && j + (int)__builtin_ctzll(mask) < first;
            count += __popcll(mask);
        }
        if (earlier || count == 0) continue;
        if (count * per > MANY) {
            if (lane == 0) l.many[atomicAdd(&l.n_many, 1)] = tl;      // (their order does not matter: each is a sum of its own)
            continue;
        }
        for (int c0 = 0; c0 < cpr; c0 += 64) {
            const int chunks = min(cpr - c0, 64), g = 64 / chunks, y = lane / chunks, c = chunk_at<WIDE>(c0 + lane % chunks, a.d);
            float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            for (int j = first & ~63; j < m; j += 64) {
                const bool in = j + lane < m && l.tok[min(j + lane, m - 1)] == tl;
                const unsigned long long mask = __ballot(in);
                if (mask == 0) continue;
                __builtin_amdgcn_wave_barrier();
                if (in) l.mine[wave][__popcll(mask & ((1ull << lane) - 1))] = l.pos[j + lane];
                __builtin_amdgcn_wave_barrier();
                if (y < g) few_rows<T, WIDE>(a, l.mine[wave], (int)__popcll(mask) * per, y, g, c, s);
            }
            __builtin_amdgcn_wave_barrier();
            if (y < g)
#pragma unroll
                for (int x = 0; x < 8; ++x)
                    if (c + x >= 8 * c0) sums[y * 8 * chunks + c - 8 * c0 + x] = s[x];
            __builtin_amdgcn_wave_barrier();
            for (int z = lane; z < 8 * chunks; z += 64) {
                float r = sums[z];
                for (int q = 1; q < g; ++q) r += sums[q * 8 * chunks + z];
                if (8 * c0 + z < a.d) put_one<T>(a, t0 + (tl << bits), 8 * c0 + z, r);
            }
        }
    }
    __syncthreads();
    const int many = l.n_many;
    for (int i = 0; i < many; ++i) {
        const unsigned token = t0 + (l.many[i] << bits);
        __syncthreads();
        few_whole<T, WIDE>(a, token, few_collect(a, token, 32, l), l);
    }
}

__global__ __launch_bounds__(256) void k_clear(void* table, size_t bytes) { clear(table, bytes, (size_t)blockIdx.x * 256 + threadIdx.x, (size_t)gridDim.x * 256); }

struct Plan {
    long rows, pieces;
    int len, passes, bits, tiles;
    bool few;
    size_t sorted, other, counts, totals, part, bytes;      // offsets into the workspace
};

Plan plan(long n, long per, long v, int d) {
    Plan p{};
    p.rows = n * per;
    // pieces: enough threads (a thread = 8 columns of a piece) to fill the chip's 256 x 4 SIMDs a few waves deep; 16 rows at least, so that partial sums stay few
    const long cpr = (d + 7) / 8;
    long len = (p.rows * cpr + 131071) / 131072;
    len = len < 16 ? 16 : len > 256 ? 256 : (len + 7) & ~7L;
    p.len = (int)len;
    p.pieces = (p.rows + len - 1) / len;
    int all = 1;
    while ((v >> all) != 0) ++all;               // keys are 0 .. v
    p.passes = (all + 8) / 9;
    p.bits = (all + p.passes - 1) / p.passes;
    p.tiles = n > SMALL ? (int)((n + TILE - 1) / TILE) : 0;
    // (a token's rows are one workgroup's work there: not where few tokens share much)
    p.few = n > 0 && n <= FEW && p.rows <= FEW_ROWS && v <= 131072 && p.rows * d <= FEW_ELEMENTS && p.rows * d <= FEW_SHARE * v;
    if (p.few || n == 0) {
        p.bytes = 0;
        return p;
    }
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t was = at; at += (bytes + 255) & ~(size_t)255; return was; };
    p.sorted = take((size_t)n * sizeof(Entry));
    p.other = take(p.tiles ? (size_t)n * sizeof(Entry) : 0);
    p.counts = take((size_t)p.tiles << (p.bits + 2));
    p.totals = take(BINS * 4);
    p.part = take((size_t)p.pieces * 2 * 8 * cpr * 4);
    p.bytes = at;
    return p;
}

template <int T> hipError_t lookup_backward(const LookupGrad& a, hipStream_t s) {
    const Plan p = plan(a.n, a.per, a.v, a.d);
    char* ws = static_cast<char*>(a.ws);
    auto u = [&](size_t at) { return reinterpret_cast<unsigned*>(ws + at); };
    Entry *sorted = reinterpret_cast<Entry*>(ws + p.sorted), *other = reinterpret_cast<Entry*>(ws + p.other);
    const size_t zero = (size_t)a.v * a.d * Bytes<T>::v;
    if (p.few) {
        // one workgroup a compute unit: 512 (1 024) of them took 16 (26) us instead of 10.5 for 4 096 of 4 096 x 48, 43 (60) instead of 38 for 10 762 of 56 940 x 69
        const bool alone = a.v <= 256;
        const dim3 grid(alone ? (unsigned)a.v : 256);
        if (a.d >= 8) hipLaunchKernelGGL((k_lookup_few<T, true>), grid, dim3(1024), 0, s, a, alone ? 32 : 8);
        else hipLaunchKernelGGL((k_lookup_few<T, false>), grid, dim3(1024), 0, s, a, alone ? 32 : 8);
        return hipGetLastError();
    }
    if (a.n == 0 || p.tiles == 0) {
        // a table of up to 64 KB is cleared by the sorting workgroup, a larger one by a launch of its own
        const bool own = a.n > 0 && zero <= 65536;
        if (!own) hipLaunchKernelGGL(k_clear, dim3((unsigned)(zero / 4096 < 4095 ? zero / 4096 + 1 : 4096)), dim3(256), 0, s, a.dtable, zero);
        if (a.n == 0) return hipGetLastError();
        hipLaunchKernelGGL(k_sort_small, dim3(1), dim3(1024), 0, s, a, p.passes, p.bits, sorted, own ? zero : 0);
    } else {
        const Entry* from = nullptr;
        for (int pass = 0; pass < p.passes; ++pass) {
            Entry* to = ((p.passes - 1 - pass) & 1) != 0 ? other : sorted;      // the last pass ends in `sorted`
            hipLaunchKernelGGL(k_sort_count, dim3(p.tiles), dim3(256), 0, s, a, from, pass * p.bits, p.bits, u(p.counts), pass == 0 ? zero : 0);
            hipLaunchKernelGGL(k_sort_scan, dim3(1u << p.bits), dim3(256), 0, s, u(p.counts), p.tiles, u(p.totals));
            hipLaunchKernelGGL(k_sort_scatter, dim3(p.tiles), dim3(256), 0, s, a, from, pass * p.bits, p.bits, u(p.counts), u(p.totals), to);
            from = to;
        }
    }
    const long threads = p.pieces * ((a.d + 7) / 8);
    float* part = reinterpret_cast<float*>(ws + p.part);
    const dim3 grid((unsigned)((threads + 255) / 256));
    if (a.d >= 8) hipLaunchKernelGGL((k_lookup_sum<T, true>), grid, dim3(256), 0, s, a, sorted, p.pieces, p.len, part);
    else hipLaunchKernelGGL((k_lookup_sum<T, false>), grid, dim3(256), 0, s, a, sorted, p.pieces, p.len, part);
    if (p.pieces > 1) hipLaunchKernelGGL((k_lookup_join<T>), dim3((unsigned)((p.pieces + 3) / 4)), dim3(256), 0, s, a, sorted, p.pieces, p.len, part);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_lookup(int type, const Lookup& a, hipStream_t s) {
    const long blocks = (a.n * a.per * ((a.d + 7) / 8) + 255) / 256;
    const dim3 g((unsigned)(blocks < 16384 ? blocks : 16384)), b(256);
    if (type == LT_F32) hipLaunchKernelGGL((k_lookup<LT_F32>), g, b, 0, s, a);
    else if (type == LT_BF16) hipLaunchKernelGGL((k_lookup<LT_BF16>), g, b, 0, s, a);
    else hipLaunchKernelGGL((k_lookup<LT_F16>), g, b, 0, s, a);
    return hipGetLastError();
}

size_t lookup_backward_bytes(long n, long per, long v, int d) { return plan(n, per, v, d).bytes; }

hipError_t launch_lookup_backward(int type, const LookupGrad& a, hipStream_t s) {
    return type == LT_F32 ? lookup_backward<LT_F32>(a, s) : type == LT_BF16 ? lookup_backward<LT_BF16>(a, s) : lookup_backward<LT_F16>(a, s);
}

}  // namespace ibl
