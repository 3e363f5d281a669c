// Linear layers and 1x1 convolutions in 8-bit integers, a scale per token and per output channel (gfx950).  The formulas
// stand in include/ddcn_hip.h.
//
//   prepare_*    x (any strides) -> codes and the tokens' scales; workgroups behind those of the tokens repack the weights
//   gemm8        (many tokens) codes x weights on v_mfma_i32_16x16x64_i8, operands global -> LDS by DMA through a ring of K
//                steps; exact int32 sums, scales + bias + ReLU in the epilogue, or int32 partial sums where K is split
//   direct8      (from 17 tokens on, see plan_of) codes straight into the MFMA's registers, weights from the caller's rows
//   gemv8        (up to 16) a wave per channel streams its weights once, v_dot4_i32_i8; up to 4 tokens it rounds them too
//   finish       sums of the partial sums, epilogue
//
// Codes and repacked weights are stored as [k / 16][token or channel][16]: sixteen consecutive k of one row are one operand
// fragment of the MFMA, rows follow each other.  A DMA request of 64 lanes is then 1 KB in a row, the LDS image needs no
// swizzle, and both preparing kernels write whole lines.  k is padded with zeros to whole K steps of 64.
#include "ddcn_elem.h"

namespace ddcn {
namespace {

typedef __attribute__((ext_vector_type(4))) int i32x4;

constexpr int kMaxK = 131072;          // k * 127 * 128 stays below 2^31
// Tokens of one pass: offsets within four rows of chunks fit 31 bits, and a workgroup of 256 threads for each of them makes
// a grid of 2^31 threads (below 2^32)
constexpr long long kPassTokens = 1LL << 23;

struct Int8Args {
    const void *x;
    u32x4 *q;                          // codes [chunks][ldq]
    float *scale;                      // [tokens of the pass]
    signed char *q_rows;               // ddcn_int8_quantize: codes [token][ldq] instead
    const signed char *w;
    u32x4 *wp;                         // repacked weights [chunks][channels]
    const float *w_scale, *bias;
    void *y;
    int *part;                         // partial sums [split][rows][cols]
    long long t0;                      // first token of the pass
    long long si, sh, sw, sk, ldq, ldw;
    int tokens;                        // of the pass
    int plane, cols;                   // of an image
    int k, chunks, channels, relu;     // chunks: of 16 k, whole K steps
    int prep_blocks;                   // workgroups of the tokens; the rest repack weights
    int splits, steps_per;             // of K, and K steps of one
};

// Workgroups round-robin over the 8 XCDs by launch index: give each XCD a contiguous run of tiles (bijective)
__device__ __forceinline__ int xcd_logical(int b, int total)
{
    const int q = total / 8, r = total % 8, xcd = b % 8, k = b / 8;
    return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + k;
}

// first element of token t (of the pass) in x
__device__ __forceinline__ long long token_base(const Int8Args &a, int t)
{
    const unsigned u = (unsigned)(a.t0 + t), img = u / (unsigned)a.plane, p = u - img * (unsigned)a.plane;
    const unsigned h = p / (unsigned)a.cols;
    return img * a.si + h * a.sh + (p - h * (unsigned)a.cols) * a.sw;
}

// Scale and factor from the largest |x| of a token, given as its bits (ordered as the numbers are, NaN on top).  Factor 0
// marks a token with a NaN or an infinity: its codes are 0 and its scale is NaN.
__device__ __forceinline__ void token_scale(unsigned top, float &scale, float &factor)
{
    constexpr unsigned kLeast = 0x0F800000u, kInf = 0x7F800000u;      // 2^-96
    const float m = __uint_as_float(max(top, kLeast));
    scale = top >= kInf ? __uint_as_float(0x7FC00000u) : m / 127.f;
    factor = top >= kInf ? 0.f : 127.f / m;
}
__device__ __forceinline__ unsigned bits_of(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// Adding 1.5 * 2^23 rounds to the nearest even whole number and leaves it in the low bits: the product is rounded to fp32
// first, as the code is defined.  (NaN and infinity times 0 leave other bits there: masked by `fine`.)
__device__ __forceinline__ unsigned code(float x, float factor)
{
#pragma clang fp contract(off)
    const float v = x * factor;
    return __float_as_uint(v + 12582912.f) & 255u;
}
__device__ __forceinline__ u32x4 pack16(const float (&x)[16], float factor)
{
    u32x4 r;
#pragma unroll
    for (int d = 0; d < 4; ++d)
        r[d] = code(x[4 * d], factor) | code(x[4 * d + 1], factor) << 8 | code(x[4 * d + 2], factor) << 16 | code(x[4 * d + 3], factor) << 24;
    const unsigned fine = factor > 0.f ? ~0u : 0u;
    return u32x4{r[0] & fine, r[1] & fine, r[2] & fine, r[3] & fine};
}

// ---------------------------------------------------------------- weights
// 16 weight bytes from k on, zero behind the row's kk bytes
__device__ __forceinline__ u32x4 weight_chunk(const signed char *row, int k, int kk, bool wide)
{
    if (k >= kk) return u32x4{0u, 0u, 0u, 0u};
    if (wide && k + 16 <= kk) return *(const u32x4 *)(row + k);
    unsigned u[4] = {0u, 0u, 0u, 0u};
    for (int e = 0; e < 16; ++e)
        if (k + e < kk) u[e >> 2] |= (unsigned)(unsigned char)row[k + e] << (8 * (e & 3));
    return u32x4{u[0], u[1], u[2], u[3]};
}
__device__ __forceinline__ bool wide_rows(const Int8Args &a) { return (((unsigned long long)a.w | (unsigned long long)a.ldw) & 15) == 0; }

// A wave moves 8 rows x 8 chunks: 128-byte lines on both sides
__device__ __forceinline__ void repack_weights(const Int8Args &a, int block, int blocks)
{
    const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
    const int across = (a.chunks + 7) / 8, items = (a.channels + 7) / 8 * across;
    const bool wide = wide_rows(a);
    for (int i = block * waves + (threadIdx.x >> 6); i < items; i += blocks * waves) {
        const int n = i / across * 8 + (lane & 7), c = i % across * 8 + (lane >> 3);
        if (n < a.channels && c < a.chunks)
            a.wp[(long long)c * a.channels + n] = weight_chunk(a.w + n * a.ldw, c * 16, a.k, wide);
    }
}

// ---------------------------------------------------------------- tokens
__device__ __forceinline__ void store_chunk(const Int8Args &a, int t, int c, u32x4 v)
{
    if (!a.q_rows) {
        a.q[(long long)c * a.ldq + t] = v;
    } else {                                               // rows of bytes: only what exists
        signed char *row = a.q_rows + (a.t0 + t) * a.ldq;
        for (int e = 0; e < 16; ++e)
            if (c * 16 + e < a.ldq) row[c * 16 + e] = (signed char)(v[e >> 2] >> (8 * (e & 3)));
    }
}

template <int DT> __device__ __forceinline__ void load_16(const Int8Args &a, long long base, int k, bool vec, float (&x)[16])
{
    if (vec && k + 16 <= a.k) {
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            float f[4];
            if (DT == DDCN_F32) load_four<DT>(a.x, base + k + 4 * d, f);
            else if (d & 1) continue;
            else {
                const u32x4 u = *(const u32x4 *)((const bf16_t *)a.x + base + k + 4 * d);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[4 * d + 2 * e] = DT == DDCN_BF16 ? BF16::lo(u[e]) : F16::lo(u[e]);
                    x[4 * d + 2 * e + 1] = DT == DDCN_BF16 ? BF16::hi(u[e]) : F16::hi(u[e]);
                }
                continue;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * d + e] = f[e];
        }
        return;
    }
    if (k + 16 <= a.k) {
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = load_one<DT>(a.x, base + (k + e) * a.sk);
    } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = k + e < a.k ? load_one<DT>(a.x, base + (k + e) * a.sk) : 0.f;
    }
}

// sk == 1, a row of x per token: 16 consecutive values per lane and turn, up to I turns held in registers (more are read
// again).  W > 1: W waves per token.  W == 1: 2^lanes_log lanes per token (all 64 if I > 1), 512 threads, whose codes meet in
// LDS and leave as whole lines -- eight tokens a workgroup at least (60000 x 2048 bf16: 63 us, 5.8 TB/s; a wave storing the 16
// bytes of each chunk by itself 93; 60000 x 64: 4.6 us, 24 with a wave for each token).
template <int DT, int W, int I> __global__ __launch_bounds__(W == 1 ? 512 : 64 * W) void prepare_rows_kernel(const Int8Args a, int lanes_log)
{
    if ((int)blockIdx.x >= a.prep_blocks) return repack_weights(a, blockIdx.x - a.prep_blocks, gridDim.x - a.prep_blocks);
    if (W > 1 || I > 1) lanes_log = 6;
    const int lanes = 1 << lanes_log, tokens = W == 1 ? 512 >> lanes_log : 1, turn = lanes * W;        // turn: chunks of one
    __shared__ unsigned tops[4];
    __shared__ u32x4 lines[W == 1 ? I * 512 : 1];
    const int j = W == 1 ? threadIdx.x >> lanes_log : 0, first = threadIdx.x & (turn - 1);
    const int t_first = xcd_logical(blockIdx.x, a.prep_blocks) * tokens, t = t_first + j;
    const bool live = t < a.tokens;
    const long long base = live ? token_base(a, t) : 0;
    constexpr int kAlign = DT == DDCN_F32 ? 4 : 8;
    const bool vec = (base & (kAlign - 1)) == 0 && ((unsigned long long)a.x & 15) == 0;
    float x[I][16];
    unsigned top = 0;
    if (live) {
#pragma unroll
        for (int i = 0; i < I; ++i)
            if (first + i * turn < a.chunks) load_16<DT>(a, base, (first + i * turn) * 16, vec, x[i]);
#pragma unroll
        for (int i = 0; i < I; ++i)
            if (first + i * turn < a.chunks)
#pragma unroll
                for (int e = 0; e < 16; ++e) top = max(top, bits_of(x[i][e]));
        for (int c = first + I * turn; c < a.chunks; c += turn) {
            float z[16];
            load_16<DT>(a, base, c * 16, vec, z);
#pragma unroll
            for (int e = 0; e < 16; ++e) top = max(top, bits_of(z[e]));
        }
    }
    for (int d = lanes >> 1; d; d >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, d));
    if (W > 1) {
        if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
        __syncthreads();
        top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
    }
    float scale, factor;
    token_scale(top, scale, factor);
    if (live && first == 0) a.scale[a.q_rows ? a.t0 + t : t] = scale;
    if (W == 1 && !a.q_rows) {
        // chunk c of token j in place j ^ (c % 8) of its line
#pragma unroll
        for (int i = 0; i < I; ++i) {
            const int c = first + i * turn;
            if (live && c < a.chunks) lines[c * tokens + (j ^ (c & 7))] = pack16(x[i], factor);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < a.chunks * tokens; i += 512) {
            const int c = i >> (9 - lanes_log), to = t_first + ((i & (tokens - 1)) ^ (c & 7));
            if (to < a.tokens) a.q[(long long)c * a.ldq + to] = lines[i];
        }
        return;
    }
    if (!live) return;
#pragma unroll
    for (int i = 0; i < I; ++i)
        if (first + i * turn < a.chunks) store_chunk(a, t, first + i * turn, pack16(x[i], factor));
    for (int c = first + I * turn; c < a.chunks; c += turn) {
        float z[16];
        load_16<DT>(a, base, c * 16, vec, z);
        store_chunk(a, t, c, pack16(z, factor));
    }
}

// Sixteen values of a chunk as they are stored: 16-bit ones in pairs
template <int DT> struct Raw {
    static constexpr int N = DT == DDCN_F32 ? 16 : 8;
    unsigned u[N];
};
template <int DT> __device__ __forceinline__ Raw<DT> paired(const unsigned (&v)[16])
{
    Raw<DT> r;
#pragma unroll
    for (int e = 0; e < Raw<DT>::N; ++e) r.u[e] = DT == DDCN_F32 ? v[e] : v[2 * e] | v[2 * e + 1] << 16;
    return r;
}
template <int DT> __device__ __forceinline__ unsigned raw_one(const void *p)
{
    return DT == DDCN_F32 ? *(const unsigned *)p : (unsigned)*(const bf16_t *)p;
}
// any address and any end of k
template <int DT> __device__ __forceinline__ Raw<DT> load_raw(const Int8Args &a, long long base, int k)
{
    constexpr int kSize = DT == DDCN_F32 ? 4 : 2;
    unsigned v[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = k + e < a.k ? raw_one<DT>((const char *)a.x + (base + (k + e) * a.sk) * kSize) : 0u;
    return paired<DT>(v);
}
// `from` is the wave's address of the first value, `off` the lane's distance from it: no address arithmetic per load
template <int DT> __device__ __forceinline__ Raw<DT> load_raw_near(const char *from, long long step, unsigned off)
{
    unsigned v[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = raw_one<DT>(from + e * step + off);
    return paired<DT>(v);
}
// the larger of `top` and the chunk's magnitudes, on their bits (16-bit formats are ordered by them too, half by half)
template <int DT> __device__ __forceinline__ unsigned top_raw(const Raw<DT> &r, unsigned top)
{
    typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;
#pragma unroll
    for (int e = 0; e < Raw<DT>::N; ++e)
        if (DT == DDCN_F32) top = max(top, r.u[e] & 0x7FFFFFFFu);
        else top = __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2, top), __builtin_bit_cast(u16x2, r.u[e] & 0x7FFF7FFFu)));
    return top;
}
// fp32 bits of what top_raw gives
template <int DT> __device__ __forceinline__ unsigned top_bits(unsigned top)
{
    if (DT == DDCN_F32) return top;
    const unsigned one = max(top & 0xFFFFu, top >> 16);
    return DT == DDCN_BF16 ? one << 16 : __float_as_uint(F16::one((bf16_t)one));
}
template <int DT> __device__ __forceinline__ u32x4 pack_raw(const Raw<DT> &r, float factor)
{
    float x[16];
#pragma unroll
    for (int e = 0; e < Raw<DT>::N; ++e) {
        if (DT == DDCN_F32) x[e] = __uint_as_float(r.u[e]);
        else {
            x[2 * e] = DT == DDCN_BF16 ? BF16::lo(r.u[e]) : F16::lo(r.u[e]);
            x[2 * e + 1] = DT == DDCN_BF16 ? BF16::hi(r.u[e]) : F16::hi(r.u[e]);
        }
    }
    return pack16(x, factor);
}

// Any strides, lanes along the tokens: 32 tokens per workgroup; a wave takes two chunks of 16 channels at a time (one per
// half), I such pairs held in registers as they came (more are read again).  16-bit values in pairs leave room for two
// workgroups of 1024 on a CU: one loads while the other rounds and stores.  Bound by HBM: 32768 x 2048 bf16 in 48 us (201 MB,
// 4.2 TB/s); two pixels to a load, 64 tokens to a workgroup takes 49, and more where pixels are few.
template <int DT, int NT, int I> __global__ __launch_bounds__(NT, DT != DDCN_F32 && NT == 1024 ? 8 : 4) void prepare_map_kernel(const Int8Args a)
{
    if ((int)blockIdx.x >= a.prep_blocks) return repack_weights(a, blockIdx.x - a.prep_blocks, gridDim.x - a.prep_blocks);
    constexpr int kWaves = NT / 64, kSize = DT == DDCN_F32 ? 4 : 2;
    __shared__ unsigned tops[kWaves][32];
    const int tl = threadIdx.x & 31, high = (threadIdx.x >> 5) & 1, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t_first = xcd_logical(blockIdx.x, a.prep_blocks) * 32;    // neighbours share lines of x, and an L2
    const int t = t_first + tl;
    const bool live = t < a.tokens;
    const long long start = token_base(a, t_first), base = live ? token_base(a, t) : start;
    // the lane's distance from the workgroup's first token, with the half's 16 channels: within 32 bits nearly always
    const long long apart = (base - start + high * 16 * a.sk) * kSize;
    const bool near = __all(apart >= 0 && apart < (1LL << 31));
    const char *from = (const char *)a.x + start * kSize;
    auto load = [&](int pair) {
        if (near && (pair + 1) * 32 <= a.k) return load_raw_near<DT>(from + pair * 32 * a.sk * kSize, a.sk * kSize, (unsigned)apart);
        return load_raw<DT>(a, base, (pair * 2 + high) * 16);
    };
    const int pairs = (a.chunks + 1) / 2;
    Raw<DT> x[I];
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < I; ++i)
        if (wave + i * kWaves < pairs) x[i] = load(wave + i * kWaves);
#pragma unroll
    for (int i = 0; i < I; ++i)
        if (wave + i * kWaves < pairs) top = top_raw<DT>(x[i], top);
    for (int p = wave + I * kWaves; p < pairs; p += kWaves) top = top_raw<DT>(load(p), top);
    top = top_bits<DT>(top);
    top = max(top, (unsigned)__shfl_xor((int)top, 32));
    if (high == 0) tops[wave][tl] = top;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) top = max(top, tops[w][tl]);
    float scale, factor;
    token_scale(top, scale, factor);
    auto store = [&](int pair, const Raw<DT> &r) {
        if (live && pair * 2 + high < a.chunks) store_chunk(a, t, pair * 2 + high, pack_raw<DT>(r, factor));
    };
#pragma unroll
    for (int i = 0; i < I; ++i)
        if (wave + i * kWaves < pairs) store(wave + i * kWaves, x[i]);
    for (int p = wave + I * kWaves; p < pairs; p += kWaves) store(p, load(p));
    if (live && wave == 0 && high == 0) a.scale[a.q_rows ? a.t0 + t : t] = scale;
}

// ---------------------------------------------------------------- epilogue
__device__ __forceinline__ float finished(const Int8Args &a, int sum, float st, float sn, float bias)
{
#pragma clang fp contract(off)
    float v = (float)sum * (st * sn);
    if (a.bias) v = v + bias;
    return a.relu && v < 0.f ? 0.f : v;                    // a NaN stays
}
// where token t (of the pass), channel 0 lies in y, and the stride of the channels
template <bool NCHW> __device__ __forceinline__ long long out_base(const Int8Args &a, int t)
{
    const unsigned u = (unsigned)(a.t0 + t);
    if (!NCHW) return (long long)u * a.channels;
    const unsigned img = u / (unsigned)a.plane;
    return (long long)img * a.channels * a.plane + (u - img * (unsigned)a.plane);
}

// ---------------------------------------------------------------- product
// N requests of 16 bytes per lane from `from` (`bytes` readable there), to LDS STEP bytes apart
template <int N, int STEP> __device__ __forceinline__ void dma(const u32x4 *from, unsigned bytes, char *to, const unsigned *off)
{
    const __amdgpu_buffer_rsrc_t r = uniform_rsrc(from, bytes);
#pragma unroll
    for (int i = 0; i < N; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void *)(to + i * STEP), 16, off[i], 0, 0, 0);
}

__device__ __forceinline__ i32x4 mfma8(u32x4 a, u32x4 b, i32x4 c)
{
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

// Rows of the tile run along the registers of the result, columns along its lanes; the rows are what is contiguous in y --
// tokens for nchw (columns: channels), channels otherwise (columns: tokens) -- so that a lane ends with runs of y in its
// registers and stores 16 bytes at a time (stores of single 16-bit elements cost 65 cycles each: 28 us of a 256-tile round).
// For that, LDS slot s of a 32-row group holds row `row_of(s)`: a lane's results of two neighbouring 16-row tiles are then
// eight consecutive rows (16-bit results; four of one tile for fp32).
// Tile 2*MI*32 rows x 64*NWN columns, 2 x NWN waves of MI*32 x 64.  A ring of NS K steps (64 k each) in LDS, filled by DMA:
// the request of step s + NS goes into the stage that step s has left.  One barrier per step, between the two halves of its
// MFMAs: fragments are read one half ahead of their use.
template <bool PAIRS> __device__ __forceinline__ int row_of(int s)
{
    // slot = tile * 16 + quad * 4 + e  ->  row = quad * 8 + tile * 4 + e
    return PAIRS ? (s & ~31) | ((s >> 2) & 3) << 3 | ((s >> 4) & 1) << 2 | (s & 3) : s;
}

// N consecutive values of y; the address is aligned to its elements only
template <int DT, int N> __device__ __forceinline__ void store_run(void *y, long long at, const float (&v)[N])
{
    if (DT == DDCN_F32) {
        struct __attribute__((packed, aligned(4))) Run {
            float f[N];
        } r;
#pragma unroll
        for (int e = 0; e < N; ++e) r.f[e] = v[e];
        *(Run *)((float *)y + at) = r;
    } else {
        struct __attribute__((packed, aligned(2))) Run {
            unsigned u[N / 2];
        } r;
#pragma unroll
        for (int e = 0; e < N / 2; ++e)
            r.u[e] = DT == DDCN_BF16 ? BF16::pack2(v[2 * e], v[2 * e + 1]) : F16::pack2(v[2 * e], v[2 * e + 1]);
        *(Run *)((bf16_t *)y + at) = r;
    }
}

template <int DT, bool NCHW, bool PART, int MI, int NWN, int NS>
__global__ __launch_bounds__(128 * NWN, 4) void gemm8_kernel(const Int8Args a)
{
    constexpr int NT = 128 * NWN, NWAVES = NT / 64, BR = 2 * MI * 32, BC = 64 * NWN;
    constexpr int RR = BR * 4 / NT, RC = BC * 4 / NT;      // requests per thread and step
    constexpr int STAGE = BR * 4 + BC * 4;                 // 16-byte chunks of a stage
    constexpr bool PAIRS = !PART && DT != DDCN_F32;
    extern __shared__ u32x4 ring[];
    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wr = wave / NWN, wc = wave % NWN;
    const int rows = NCHW ? a.tokens : a.channels, cols = NCHW ? a.channels : a.tokens;
    const u32x4 *R = NCHW ? a.q : a.wp, *C = NCHW ? a.wp : a.q;
    const long long ldr = NCHW ? a.ldq : a.channels, ldc = NCHW ? a.channels : a.ldq;
    const int tiles_r = (rows + BR - 1) / BR, tiles_c = (cols + BC - 1) / BC;
    // Whole K: neighbours share the tile of tokens, the larger operand.  Split: an XCD takes one piece of K (the splits are
    // mostly a power of two) and its L2 reads that piece of both operands alone.
    const int L = PART ? blockIdx.x / a.splits : xcd_logical(blockIdx.x, tiles_r * tiles_c), split = PART ? blockIdx.x % a.splits : 0;
    const int r0 = (NCHW ? L / tiles_c : L % tiles_r) * BR, c0 = (NCHW ? L % tiles_c : L / tiles_r) * BC;
    const int first = split * a.steps_per, steps = min(a.steps_per, a.chunks / 4 - first);

    unsigned off_r[RR], off_c[RC];
#pragma unroll
    for (int i = 0; i < RR; ++i) {
        const int q = (i * NWAVES + wave) * 64 + lane, row = row_of<PAIRS>(q % BR);
        off_r[i] = r0 + row < rows ? (unsigned)((q / BR) * ldr + row) * 16u : DMA_OOB;
    }
#pragma unroll
    for (int i = 0; i < RC; ++i) {
        const int q = (i * NWAVES + wave) * 64 + lane, col = q % BC;
        off_c[i] = c0 + col < cols ? (unsigned)((q / BC) * ldc + col) * 16u : DMA_OOB;
    }
    const u32x4 *pr = R + (long long)first * 4 * ldr + r0, *pc = C + (long long)first * 4 * ldc + c0;
    const unsigned lim_r = (unsigned)(4 * ldr - r0) * 16u, lim_c = (unsigned)(4 * ldc - c0) * 16u;
    auto request = [&](int s) {
        char *base = (char *)(ring + (s % NS) * STAGE) + wave * 1024;
        dma<RR, NWAVES * 1024>(pr + (long long)s * 4 * ldr, lim_r, base, off_r);
        dma<RC, NWAVES * 1024>(pc + (long long)s * 4 * ldc, lim_c, base + BR * 64, off_c);
    };

    constexpr int RT = 2 * MI;                             // 16-row tiles of a wave
    i32x4 acc[RT][4];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
    const int r16 = lane & 15, kc = lane >> 4;
    auto read_r = [&](int s, int h, u32x4 (&f)[MI]) {
        const u32x4 *st = ring + (s % NS) * STAGE + kc * BR + wr * (MI * 32) + h * (MI * 16) + r16;
#pragma unroll
        for (int i = 0; i < MI; ++i) f[i] = st[i * 16];
    };
    auto read_c = [&](int s, u32x4 (&f)[4]) {
        const u32x4 *st = ring + (s % NS) * STAGE + BR * 4 + kc * BC + wc * 64 + r16;
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = st[j * 16];
    };
    auto mfmas = [&](int h, const u32x4 (&fr)[MI], const u32x4 (&fc)[4]) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[h * MI + i][j] = mfma8(fr[i], fc[j], acc[h * MI + i][j]);
    };
    // this wave's LDS reads are done and all but its `younger` youngest steps have landed
    auto wait_but = [&](int younger) {
        if (NS > 3 && younger >= 3) __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(3 * (RR + RC)));
        else if (younger == 2) __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(2 * (RR + RC)));
        else if (younger == 1) __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(RR + RC));
        else __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(0));
    };
    static_assert(NS <= 4 && 3 * (RR + RC) < 64, "vmcnt is 6 bits and wait_but knows up to 3 steps in flight");
    u32x4 f0[MI], f1[MI], fx[4], fy[4];
    auto step = [&](int s, u32x4 (&fc)[4], u32x4 (&fn)[4]) {
        read_r(s, 1, f1);
        __builtin_amdgcn_sched_barrier(0);
        mfmas(0, f0, fc);
        __builtin_amdgcn_sched_barrier(0);
        if (s + 1 < steps) {
            wait_but(min(NS - 2, steps - 2 - s));
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
            if (s + NS < steps) request(s + NS);
            read_c(s + 1, fn);
            read_r(s + 1, 0, f0);
            __builtin_amdgcn_sched_barrier(0);
        }
        mfmas(1, f1, fc);
        __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int s = 0; s < NS; ++s)
        if (s < steps) request(s);
    wait_but(min(NS - 1, steps - 1));
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    read_c(0, fx);
    read_r(0, 0, f0);
    for (int s = 0; s < steps; s += 2) {
        step(s, fx, fy);
        if (s + 1 < steps) step(s + 1, fy, fx);
    }

    // lane l holds slots 4 * (l / 16) + e, column l % 16 of each 16 x 16 tile: runs of N consecutive rows
    constexpr int N = PAIRS ? 8 : 4, T = N / 4;
    const int row0 = r0 + wr * (MI * 32) + kc * N, col0 = c0 + wc * 64 + r16;
    float sc[4], bc[4];
    if (!PART)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int col = min(col0 + j * 16, cols - 1);
            sc[j] = NCHW ? a.w_scale[col] : a.scale[col];
            bc[j] = NCHW && a.bias ? a.bias[col] : 0.f;
        }
    if (PART) {
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const int row = row0 + i * 16, live = min(rows - row, 4);
            int *part = a.part + (long long)split * rows * cols + row;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int col = col0 + j * 16;
                if (col >= cols || live <= 0) continue;
                int *to = part + (long long)col * rows;
                if (live == 4 && (rows & 3) == 0) *(i32x4 *)to = acc[i][j];
                else
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (e < live) to[e] = acc[i][j][e];
            }
        }
        return;
    }
    constexpr int G = RT / T;                              // runs of a lane and column
    float sr[G][N], br[G][N];
    long long base[G];                                     // the run's place in y, without its column
    unsigned place[G];                                     // and in its image (nchw)
    bool whole[G];                                         // all of it exists, in one image
#pragma unroll
    for (int g = 0; g < G; ++g) {
        const int row = row0 + g * T * 16;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const int at = min(row + e, rows - 1);
            sr[g][e] = NCHW ? a.scale[at] : a.w_scale[at];
            br[g][e] = !NCHW && a.bias ? a.bias[at] : 0.f;
        }
        const unsigned u = (unsigned)(a.t0 + row), img = NCHW ? u / (unsigned)a.plane : 0u;
        place[g] = NCHW ? u - img * (unsigned)a.plane : 0u;
        whole[g] = rows - row >= N && (!NCHW || place[g] + N <= (unsigned)a.plane);
        base[g] = NCHW ? (long long)img * a.channels * a.plane + place[g] : row;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int col = col0 + j * 16;
        const bool exists = col < cols;
        const long long off = NCHW ? (long long)col * a.plane : (a.t0 + col) * (long long)a.channels;
        float v[G][N];
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int e = 0; e < N; ++e)
                v[g][e] = finished(a, acc[g * T + e / 4][j][e & 3], NCHW ? sr[g][e] : sc[j], NCHW ? sc[j] : sr[g][e], NCHW ? bc[j] : br[g][e]);
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const int row = row0 + g * T * 16, live = rows - row;
            const long long at = base[g] + off;
            // A 16-byte store at an odd address (in 16-bit elements: every other channel of a map with an odd number of
            // pixels) takes twice as long as one at an even one.  There a run is written one element on: its own 1 .. 7 and
            // the first of the next run, which the lane 16 on holds (from the fourth sixteen on: the first sixteen's, of
            // the next g).  Its own first element is written by the run before it, where there is one in the wave and image.
            bool odd = false;
            if (PAIRS) {
                odd = exists && whole[g] && (((unsigned long long)a.y >> 1) + at & 1) != 0;
                if (__any(odd)) {
                    const float give = kc == 0 ? v[g + 1 < G ? g + 1 : g][0] : v[g][0];
                    const float next = __shfl(give, (lane + 16) & 63);
                    const bool more = !(g == G - 1 && kc == 3) && live > N && place[g] + N < (unsigned)(NCHW ? a.plane : 0x7fffffff);
                    if (odd) {
                        if ((g == 0 && kc == 0) || (NCHW && place[g] < N)) store_one<DT>(a.y, at, v[g][0]);
                        if (more) {
                            const float r[8] = {v[g][1], v[g][2], v[g][3], v[g][N > 4 ? 4 : 0], v[g][N > 4 ? 5 : 0], v[g][N > 4 ? 6 : 0], v[g][N > 4 ? 7 : 0], next};
                            store_run<DT, 8>(a.y, at + 1, r);
                        } else {
                            const float r[6] = {v[g][1], v[g][2], v[g][3], v[g][N > 4 ? 4 : 0], v[g][N > 4 ? 5 : 0], v[g][N > 4 ? 6 : 0]};
                            store_run<DT, 6>(a.y, at + 1, r);
                            store_one<DT>(a.y, at + 7, v[g][N > 4 ? 7 : 0]);
                        }
                    }
                }
            }
            if (!exists || odd || live <= 0) continue;
            if (whole[g]) store_run<DT, N>(a.y, at, v[g]);
            else
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (e < live) store_one<DT>(a.y, NCHW ? out_base<true>(a, row + e) + off : at + e, v[g][e]);
        }
    }
}

// sums [split][columns][rows] -> y, in the order of y (300 x 1024 in three pieces: 4.0 us, a launch and one round of latencies)
template <int DT, bool NCHW> __global__ __launch_bounds__(256) void finish_kernel(const Int8Args a, int splits)
{
    const int rows = NCHW ? a.tokens : a.channels, cols = NCHW ? a.channels : a.tokens;
    const long long total = (long long)rows * cols, i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    int sum = 0;
    for (int s = 0; s < splits; ++s) sum += a.part[s * total + i];
    const int col = (int)(i / rows), row = (int)(i - (long long)col * rows);
    const int tok = NCHW ? row : col, n = NCHW ? col : row;
    store_one<DT>(a.y, out_base<NCHW>(a, tok) + (NCHW ? (long long)n * a.plane : n),
                  finished(a, sum, a.scale[tok], a.w_scale[n], a.bias ? a.bias[n] : 0.f));
}

// ---------------------------------------------------------------- few tokens
// What counts is to stream the weights once, from the caller's own rows (repacking them moves as many bytes again, twice).
// 64 tokens x 16 NW channels per workgroup, and a piece of K where PART; K is dealt to the eight waves in turns of 128 k, a
// line of a weight row, two turns ahead, and nothing is shared until the waves' sums meet in LDS.  A code fragment is four
// runs of 256 bytes and goes straight into the MFMA's registers.  A weight fragment is 16 rows x 64 bytes: loaded that way
// every lane of a quarter wave touches another line, 64 line accesses for 1 KB (43 cycles of the data return path a load
// over both operands, and 300 x 12544 x 1024 took 15.3 us in place of 11.5).  So eight lanes fetch a whole line of a row,
// by DMA, into the wave's own LDS; there chunk c of row r lies in place c ^ (r % 8), which spreads eight rows over all banks.
template <int DT, bool NCHW, bool PART, int NW> __global__ __launch_bounds__(512) void direct8_kernel(const Int8Args a)
{
    constexpr bool PAIRS = !PART && DT != DDCN_F32;
    constexpr int NR = NCHW ? 4 : NW, NC = NCHW ? NW : 4;    // tiles of 16 rows (registers, contiguous in y) and columns (lanes)
    constexpr int kWaves = 8, kTurn = 2 * NW;              // requests of a turn's weights
    extern __shared__ u32x4 ring[];                        // [wave][2 turns][request][64]; after K the waves' sums
    i32x4 (*sums)[8][64] = (i32x4 (*)[8][64])ring;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, kc = lane >> 4;
    // an XCD takes a range of channels and all tokens: its L2 then reads its part of the weights alone
    const int across = (a.tokens + 63) / 64, down = (a.channels + NW * 16 - 1) / (NW * 16), L = xcd_logical(blockIdx.x, gridDim.x);
    const int t0 = L % across * 64, n0 = L / across % down * (NW * 16), split = PART ? L / (across * down) : 0;
    const int rows = NCHW ? a.tokens : a.channels, cols = NCHW ? a.channels : a.tokens;
    const int r0 = NCHW ? t0 : n0, c0 = NCHW ? n0 : t0;
    // this lane's tokens and, of each request, its weight row and chunk (clamped: what is computed for the others is not
    // stored), in bytes from the workgroup's first ones
    const char *qb = (const char *)(a.q + t0);
    const signed char *wb = a.w + n0 * a.ldw;
    const int most = min(NW * 16, a.channels - n0) - 1;    // last row
    unsigned qo[4], wo[kTurn];
#pragma unroll
    for (int i = 0; i < 4; ++i) qo[i] = (unsigned)(min(NCHW ? row_of<PAIRS>(i * 16 + r16) : i * 16 + r16, a.tokens - 1 - t0) + kc * (int)a.ldq) * 16u;
#pragma unroll
    for (int i = 0; i < kTurn; ++i) wo[i] = (unsigned)(min(i * 8 + lane / 8, most) * (int)a.ldw + ((lane ^ lane / 8) & 7) * 16);
    u32x4 *mine = ring + wave * (2 * kTurn * 64);
    int at[NW];                                            // of this lane's row in a turn's image, without its chunk
#pragma unroll
    for (int i = 0; i < NW; ++i) at[i] = (NCHW ? i * 16 + r16 : row_of<PAIRS>(i * 16 + r16)) * 8;
    // turns of this piece of K whose weights need no guard
    const int begin = PART ? split * a.steps_per : 0, full = PART ? min(begin + a.steps_per, a.k / 128) : a.k / 128;
    const bool last = !PART || split == a.splits - 1;
    i32x4 acc[NR][NC];
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int j = 0; j < NC; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
    auto mul = [&](const u32x4 (&w)[NW], const u32x4 (&q)[4]) {
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int j = 0; j < NC; ++j) acc[i][j] = NCHW ? mfma8(q[i & 3], w[j & (NW - 1)], acc[i][j]) : mfma8(w[i & (NW - 1)], q[j & 3], acc[i][j]);
    };
    u32x4 q[2][2][4];
    auto request = [&](int s, int d) {
        dma<kTurn, 1024>((const u32x4 *)(wb + s * 128), (unsigned)(most * (int)a.ldw + a.k - s * 128), (char *)(mine + d * (kTurn * 64)), wo);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) q[d][h][i] = *(const u32x4 *)(qb + ((long long)s * 8 + h * 4) * a.ldq * 16 + qo[i]);
    };
    auto consume = [&](int d, bool more) {
        __builtin_amdgcn_sched_barrier(0);
        if (more) __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(kTurn + 8));
        else __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(0));
        asm volatile("" ::: "memory");
        u32x4 w[2][NW];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < NW; ++i) w[h][i] = mine[d * (kTurn * 64) + at[i] + ((h * 4 + kc) ^ (at[i] / 8 & 7))];
#pragma unroll
        for (int h = 0; h < 2; ++h) mul(w[h], q[d][h]);
        __builtin_amdgcn_sched_barrier(0);
    };
    // While the turn after the next exists, every turn asks for one: the number of requests in flight is known, and a turn
    // waits for its own alone.  A wave reads only what it has asked for itself.
    int s = begin + wave;
    if (s + 3 * kWaves < full) {
        request(s, 0);
        request(s + kWaves, 1);
        for (; s + 3 * kWaves < full; s += 2 * kWaves)
#pragma unroll
            for (int d = 0; d < 2; ++d) {
                consume(d, true);
                request(s + (d + 2) * kWaves, d);
            }
        consume(0, true);
        consume(1, false);
        s += 2 * kWaves;
    }
    if (s < full) request(s, 0);
    if (s + kWaves < full) request(s + kWaves, 1);
    if (s < full) consume(0, s + kWaves < full);
    if (s + 2 * kWaves < full) request(s + 2 * kWaves, 0);
    if (s + kWaves < full) consume(1, s + 2 * kWaves < full);
    if (s + 2 * kWaves < full) consume(0, false);
    if (last && full * 128 < a.k && wave == (full - begin) % kWaves) {       // the end of K; the codes are padded with zeros to whole 64
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = full * 128 + h * 64;
            u32x4 w[NW], e[4];
#pragma unroll
            for (int i = 0; i < NW; ++i) w[i] = weight_chunk(wb + min(at[i] / 8, most) * a.ldw, k + kc * 16, a.k, true);
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] = k < a.k ? *(const u32x4 *)(qb + (long long)(k / 16) * a.ldq * 16 + qo[i]) : u32x4{0u, 0u, 0u, 0u};
            mul(w, e);
        }
    }
    __syncthreads();
    // the waves' sums meet in LDS, eight tiles at a time; a wave finishes two row tiles of one column tile
    constexpr int T = 2, kRows = 8 / NC, kRounds = NR / kRows, kParts = kRows / T * NC;
    static_assert(kParts == 4, "four waves finish a round, the other four the next one");
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
        if (r) __syncthreads();
#pragma unroll
        for (int i = 0; i < kRows; ++i)
#pragma unroll
            for (int j = 0; j < NC; ++j) sums[wave][i * NC + j][lane] = acc[r * kRows + i][j];
        __syncthreads();
        const int part = wave - r * kParts;
        if (part < 0 || part >= kParts) continue;
        const int i0 = part / NC * T, j = part % NC;
        i32x4 v[T] = {};
        for (int w = 0; w < kWaves; ++w)
#pragma unroll
            for (int i = 0; i < T; ++i) v[i] += sums[w][(i0 + i) * NC + j][lane];
        const int col = c0 + j * 16 + r16;
        if (col >= cols) continue;
#pragma unroll
        for (int i = 0; i < T; ++i) {
            const int row0 = r0 + (r * kRows + i0) * 16 + (PAIRS ? kc * 8 + i * 4 : i * 16 + kc * 4);
            if (PART) {
                int *to = a.part + ((long long)split * cols + col) * rows + row0;
                if (row0 + 4 <= rows && (rows & 3) == 0) *(i32x4 *)to = v[i];
                else
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (row0 + e < rows) to[e] = v[i][e];
                continue;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = row0 + e;
                if (row >= rows) continue;
                const int t = NCHW ? row : col, n = NCHW ? col : row;
                store_one<DT>(a.y, out_base<NCHW>(a, t) + (NCHW ? (long long)n * a.plane : n),
                              finished(a, v[i][e], a.scale[t], a.w_scale[n], a.bias ? a.bias[n] : 0.f));
            }
        }
    }
}

// Up to 16 tokens: a wave per channel, the weights read once, straight from the caller's rows, 16 bytes per lane and turn;
// the codes of a chunk lie next to each other.  FUSED (up to TOK = 4 tokens whose codes fit LDS): every workgroup rounds the
// tokens itself while its first weights are on their way -- one launch, no workspace; the rounding is repeated by every
// workgroup, from the caches.  1 x 12544 x 1024 fp32: 8.1 us (two launches 4.0 + 5.3), of which 2.5 would be the weights' bytes.
template <int DT, int IN, bool NCHW, int TOK, bool FUSED> __global__ __launch_bounds__(256) void gemv8_kernel(const Int8Args a)
{
    extern __shared__ u32x4 codes[];                       // FUSED: [chunk][TOK]
    __shared__ unsigned tops[4][TOK];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = min((int)blockIdx.x * 4 + wave, a.channels - 1);
    const bool wide = wide_rows(a);
    const signed char *row = a.w + n * a.ldw;
    constexpr int kAhead = 4;
    const int full = wide ? a.k / 16 : 0;                  // chunks that one wide load brings
    u32x4 ahead[kAhead];
    auto weights = [&](int c) { return *(const u32x4 *)(row + min(c, full - 1) * 16); };
    if (full)
#pragma unroll
        for (int d = 0; d < kAhead; ++d) ahead[d] = weights(lane + 64 * d);
    float scale[TOK];
    if (FUSED) {
        constexpr int kAlign = IN == DDCN_F32 ? 4 : 8;
#pragma unroll
        for (int t = 0; t < TOK; ++t) {
            const long long base = token_base(a, min(t, a.tokens - 1));
            const bool vec = a.sk == 1 && (base & (kAlign - 1)) == 0 && ((unsigned long long)a.x & 15) == 0;
            unsigned top = 0;
            for (int c = threadIdx.x; c < a.chunks; c += 256) {
                float x[16];
                load_16<IN>(a, base, c * 16, vec, x);
#pragma unroll
                for (int e = 0; e < 16; ++e) top = max(top, bits_of(x[e]));
            }
            for (int d = 32; d; d >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, d));
            if (lane == 0) tops[wave][t] = top;
        }
        __syncthreads();
#pragma unroll
        for (int t = 0; t < TOK; ++t) {
            const long long base = token_base(a, min(t, a.tokens - 1));
            const bool vec = a.sk == 1 && (base & (kAlign - 1)) == 0 && ((unsigned long long)a.x & 15) == 0;
            float factor;
            token_scale(max(max(tops[0][t], tops[1][t]), max(tops[2][t], tops[3][t])), scale[t], factor);
            for (int c = threadIdx.x; c < a.chunks; c += 256) {
                float x[16];
                load_16<IN>(a, base, c * 16, vec, x);
                codes[c * TOK + t] = pack16(x, factor);
            }
        }
        __syncthreads();
    }
    int acc[TOK] = {};
    auto dot = [&](int c, u32x4 w) {
#pragma unroll
        for (int t = 0; t < TOK; ++t) {
            const u32x4 q = FUSED ? codes[c * TOK + t] : a.q[(long long)c * a.ldq + min(t, a.tokens - 1)];
#pragma unroll
            for (int d = 0; d < 4; ++d) acc[t] = __builtin_amdgcn_sdot4((int)w[d], (int)q[d], acc[t], false);
        }
    };
    for (int c0 = 0; c0 < full; c0 += 64 * kAhead) {       // (a wave's lanes stay together: every turn loads)
#pragma unroll
        for (int d = 0; d < kAhead; ++d) {
            const int c = c0 + 64 * d + lane;
            if (c < full) dot(c, ahead[d]);
            ahead[d] = weights(c + 64 * kAhead);
        }
    }
    for (int c = full + lane; c * 16 < a.k; c += 64) dot(c, weight_chunk(row, c * 16, a.k, wide));
#pragma unroll
    for (int t = 0; t < TOK; ++t)
        for (int d = 32; d; d >>= 1) acc[t] += __shfl_xor(acc[t], d);
    // lane t writes token t
    int sum = acc[0];
    float st = FUSED ? scale[0] : a.scale[min(lane, a.tokens - 1)];
#pragma unroll
    for (int t = 1; t < TOK; ++t) {
        sum = lane == t ? acc[t] : sum;
        if (FUSED) st = lane == t ? scale[t] : st;
    }
    if (lane >= a.tokens || (int)blockIdx.x * 4 + wave >= a.channels) return;
    store_one<DT>(a.y, out_base<NCHW>(a, lane) + (NCHW ? (long long)n * a.plane : n),
                  finished(a, sum, st, a.w_scale[n], a.bias ? a.bias[n] : 0.f));
}

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// every size a kernel indexes with; the products are formed in 64 bits
int check(const ddcn_int8_geom *g, bool product)
{
    if (!g) return fail(DDCN_ERR_BAD_ARG, "geom is NULL");
    if (g->images < 0 || g->rows < 0 || g->cols < 0) return fail(DDCN_ERR_SHAPE, "negative token grid %d x %d x %d", g->images, g->rows, g->cols);
    if (g->k < 1 || g->k > kMaxK) return fail(DDCN_ERR_UNSUPPORTED, "k = %d is outside 1 .. %d", g->k, kMaxK);
    if (g->dtype < DDCN_F32 || g->dtype > DDCN_F16) return fail(DDCN_ERR_UNSUPPORTED, "dtype %d", g->dtype);
    const long long plane = (long long)g->rows * g->cols;
    if (plane >= (1LL << 31) || plane * g->images >= (1LL << 31)) return fail(DDCN_ERR_UNSUPPORTED, "2^31 tokens and more");
    if (product) {
        if (g->channels < 1 || g->channels > (1 << 20)) return fail(DDCN_ERR_SHAPE, "channels = %d is outside 1 .. 2^20", g->channels);
        if (g->ldw < g->k) return fail(DDCN_ERR_SHAPE, "weight rows of %lld bytes hold no %d values", g->ldw, g->k);
        if (g->out_dtype < DDCN_F32 || g->out_dtype > DDCN_F16) return fail(DDCN_ERR_UNSUPPORTED, "out_dtype %d", g->out_dtype);
    }
    return DDCN_OK;
}

long long tokens_of(const ddcn_int8_geom *g) { return (long long)g->images * g->rows * g->cols; }

// How a pass of `tokens` tokens is computed
struct Plan {
    int how;               // kFused, kGemv, kDirect, kTiles
    bool small;            // tiles of 64 x 64 instead of 128 x 128
    int splits, steps_per;
    size_t q_bytes, scale_bytes, w_bytes, part_bytes;
    size_t bytes() const { return q_bytes + scale_bytes + w_bytes + part_bytes; }
};

constexpr int kCUs = 256;
constexpr int kFusedTokens = 4, kGemvTokens = 16, kDirectTokens = 512;
constexpr size_t kFusedLds = 64512;       // with the maxima within the 64 KiB that need no attribute
enum { kFused, kGemv, kDirect, kTiles };

// wide: the weights' rows start on 16 bytes, and 64 of them lie within 32-bit offsets
Plan plan_of(const ddcn_int8_geom *g, long long tokens, bool wide)
{
    Plan p = {};
    const long long chunks = ceil_div(g->k, 64) * 4, steps = chunks / 4;
    p.q_bytes = round_up((size_t)(chunks * 16 * tokens), 256);
    p.scale_bytes = round_up((size_t)tokens * sizeof(float), 256);
    const int tok = tokens == 1 ? 1 : kFusedTokens;
    if (tokens <= kFusedTokens && (size_t)(chunks * 16 * tok) <= kFusedLds) {
        p.how = kFused;
        p.q_bytes = p.scale_bytes = 0;
        return p;
    }
    p.splits = 1;
    if (tokens <= kGemvTokens) {
        p.how = kGemv;
        return p;
    }
    p.how = kTiles;
    // 128 x 128 tiles, four workgroups on a CU: 18818 x 2048 x 512 takes 28 us, 32768 x 2048 x 512 37 us (256 x 256 with
    // one workgroup on a CU: 52 and 39; 256 x 128: 35 and 40).  Smaller ones where those leave a quarter of the CUs idle.
    const long long wide_tiles = ceil_div(tokens, 128) * ceil_div(g->channels, 128);
    const long long quarters = ceil_div(tokens, 64) * ceil_div(g->channels, 64);
    p.small = wide_tiles < kCUs * 3 / 4;
    const long long tiles = p.small ? quarters : wide_tiles;
    // K is split where the tiles leave CUs without work, into a power of two of pieces of 8 steps at least; long pieces once
    // more, for a second workgroup on the CU (1024 tokens x 12544 x 1024, rows at odd addresses: 56 -> 42 us with the sums
    // of the two halves; 1024 x 1024 x 1024 would take 14 instead of 8)
    long long pieces = 1;
    while (steps / (2 * pieces) >= (tiles * pieces < kCUs ? 8 : 32) && tiles * pieces < 2 * kCUs) pieces *= 2;
    // Direct: up to 512 tokens (512 x 2048 x 512: 7.7 us, tiles 8.5 + 3.6 and the weights' repacking; 512 x 25088 x 4096: 101,
    // tiles 103 at twice the tokens, and 42 of repacking), and where tiles would split K but the direct kernel's fit the
    // CUs (1024 x 12544 x 1024: 27, tiles 37 + 5 + 4; without the split tiles win: 2048 x 2048 x 512 12.5, direct 13.2).
    const bool direct = wide && (tokens <= kDirectTokens || (pieces > 1 && quarters <= kCUs));
    if (direct) {
        p.how = kDirect;
        // Its K is split from 32 turns of 128 k on where there are CUs for it, into pieces of 8 turns at least: 300 x 12544 x
        // 1024 11.5 + 4 us (whole 22), 64 x 4096 x 1024 6 + 3.4 (whole 10.5), but 64 x 2048 x 512 5.9 + 2.9 (whole 7.6).
        // Otherwise 32 channels to a workgroup instead of 64 where there are too few tiles.
        const long long turns = g->k / 128;
        pieces = turns < 32 ? 1 : kCUs / quarters < turns / 8 ? kCUs / quarters : turns / 8;
        p.small = pieces < 2 && quarters < kCUs * 3 / 4;
        if (pieces > 1) p.steps_per = (int)ceil_div(turns, pieces);
        if (pieces > 1) p.splits = (int)ceil_div(turns, p.steps_per);
    } else {
        p.w_bytes = round_up((size_t)(chunks * 16 * g->channels), 256);
        p.steps_per = (int)ceil_div(steps, pieces);
        p.splits = (int)ceil_div(steps, p.steps_per);
    }
    if (p.splits > 1) p.part_bytes = round_up((size_t)p.splits * tokens * g->channels * sizeof(int), 256);
    return p;
}

template <int DT> void launch_prepare(Int8Args &a, bool repack, hipStream_t s)
{
    // repacking: a wave moves 64 chunks; enough workgroups to take no longer than the tokens do
    const int extra = repack ? (int)(ceil_div((long long)a.channels * a.chunks, 64 * 16) < 4096 ? ceil_div((long long)a.channels * a.chunks, 64 * 16) : 4096) : 0;
    if (a.sk == 1) {
        // four waves per token for more than 4096 values, and for more than 1024 where tokens are few (300 x 2048: 3.9 us,
        // 4.4 with one wave each; 2000 x 2048: 8.9, 7.5 with one; 18818 x 4096: 59, 46 with one)
        const bool many = a.chunks > 256 || (a.chunks > 64 && a.tokens <= 4 * kCUs);
        int lanes_log = 2;                                 // whole K steps are four chunks
        while (lanes_log < 6 && a.chunks > 1 << lanes_log) ++lanes_log;
        a.prep_blocks = (int)ceil_div(a.tokens, many ? 1 : 512 >> lanes_log);
        const unsigned grid = (unsigned)(a.prep_blocks + extra);
        if (many) prepare_rows_kernel<DT, 4, 4><<<grid, 256, 0, s>>>(a, 6);
        else if (a.chunks > 128) prepare_rows_kernel<DT, 1, 4><<<grid, 512, 0, s>>>(a, 6);
        else if (a.chunks > 64) prepare_rows_kernel<DT, 1, 2><<<grid, 512, 0, s>>>(a, 6);
        else prepare_rows_kernel<DT, 1, 1><<<grid, 512, 0, s>>>(a, lanes_log);
    } else {
        a.prep_blocks = (int)ceil_div(a.tokens, 32);
        const unsigned grid = (unsigned)(a.prep_blocks + extra);
        if (a.chunks <= 8) prepare_map_kernel<DT, 256, 1><<<grid, 256, 0, s>>>(a);
        else if (a.chunks <= 32) prepare_map_kernel<DT, 1024, 1><<<grid, 1024, 0, s>>>(a);
        else if (a.chunks <= 64) prepare_map_kernel<DT, 1024, 2><<<grid, 1024, 0, s>>>(a);
        else prepare_map_kernel<DT, 1024, 4><<<grid, 1024, 0, s>>>(a);
    }
}
int run_prepare(Int8Args &a, int dtype, bool repack, hipStream_t s)
{
    if (dtype == DDCN_F32) launch_prepare<DDCN_F32>(a, repack, s);
    else if (dtype == DDCN_BF16) launch_prepare<DDCN_BF16>(a, repack, s);
    else launch_prepare<DDCN_F16>(a, repack, s);
    return check_launch("int8 prepare");
}

template <int DT, bool NCHW, bool PART, int MI, int NWN, int NS> int launch_tiles(const Int8Args &a, hipStream_t s)
{
    constexpr int BR = 2 * MI * 32, BC = 64 * NWN, kLds = NS * (BR + BC) * 64;
    static std::atomic<uint64_t> done{0};
    if (!raise_lds_limit((const void *)gemm8_kernel<DT, NCHW, PART, MI, NWN, NS>, kLds, done)) return fail(DDCN_ERR_LAUNCH, "int8 product: LDS limit");
    const long long rows = NCHW ? a.tokens : a.channels, cols = NCHW ? a.channels : a.tokens;
    gemm8_kernel<DT, NCHW, PART, MI, NWN, NS><<<(unsigned)(ceil_div(rows, BR) * ceil_div(cols, BC) * a.splits), 128 * NWN, kLds, s>>>(a);
    return check_launch("int8 product");
}
template <int DT, bool NCHW, bool PART> int launch_gemm(const Int8Args &a, const Plan &p, hipStream_t s)
{
    if (!p.small) return launch_tiles<DT, NCHW, PART, 2, 2, 2>(a, s);
    return launch_tiles<DT, NCHW, PART, 1, 1, 4>(a, s);
}
template <int DT, bool NCHW, bool PART, int NW> int launch_direct(const Int8Args &a, hipStream_t s)
{
    constexpr int kLds = NW * 32768, kChannels = NW * 16;
    static std::atomic<uint64_t> done{0};
    if (!raise_lds_limit((const void *)direct8_kernel<DT, NCHW, PART, NW>, kLds, done)) return fail(DDCN_ERR_LAUNCH, "int8 product: LDS limit");
    const long long grid = ceil_div(a.tokens, 64) * ceil_div(a.channels, kChannels) * a.splits;
    direct8_kernel<DT, NCHW, PART, NW><<<(unsigned)grid, 512, kLds, s>>>(a);
    return check_launch("int8 product");
}
template <int DT, bool NCHW> int launch_product(const Int8Args &a, const Plan &p, hipStream_t s)
{
    const unsigned waves = (unsigned)ceil_div(a.channels, 4);
    if (p.how == kGemv) gemv8_kernel<DT, DDCN_F32, NCHW, 16, false><<<waves, 256, 0, s>>>(a);
    if (p.how == kGemv) return check_launch("int8 product");
    if (p.splits == 1 && p.how == kDirect) return p.small ? launch_direct<DT, NCHW, false, 2>(a, s) : launch_direct<DT, NCHW, false, 4>(a, s);
    if (p.splits == 1) return launch_gemm<DT, NCHW, false>(a, p, s);
    const int rc = p.how == kDirect ? launch_direct<DDCN_F32, NCHW, true, 4>(a, s) : launch_gemm<DDCN_F32, NCHW, true>(a, p, s);
    if (rc != DDCN_OK) return rc;
    finish_kernel<DT, NCHW><<<(unsigned)ceil_div((long long)a.tokens * a.channels, 256), 256, 0, s>>>(a, p.splits);
    return check_launch("int8 finish");
}
template <bool NCHW> int run_product(const Int8Args &a, const Plan &p, int dtype, hipStream_t s)
{
    if (dtype == DDCN_F32) return launch_product<DDCN_F32, NCHW>(a, p, s);
    if (dtype == DDCN_BF16) return launch_product<DDCN_BF16, NCHW>(a, p, s);
    return launch_product<DDCN_F16, NCHW>(a, p, s);
}

template <int DT, int IN, bool NCHW> void launch_fused(const Int8Args &a, hipStream_t s)
{
    const unsigned waves = (unsigned)ceil_div(a.channels, 4);
    if (a.tokens == 1) gemv8_kernel<DT, IN, NCHW, 1, true><<<waves, 256, a.chunks * 16, s>>>(a);
    else gemv8_kernel<DT, IN, NCHW, kFusedTokens, true><<<waves, 256, a.chunks * 16 * kFusedTokens, s>>>(a);
}
template <int DT, bool NCHW> void launch_fused_of(const Int8Args &a, int in, hipStream_t s)
{
    if (in == DDCN_F32) launch_fused<DT, DDCN_F32, NCHW>(a, s);
    else if (in == DDCN_BF16) launch_fused<DT, DDCN_BF16, NCHW>(a, s);
    else launch_fused<DT, DDCN_F16, NCHW>(a, s);
}
template <bool NCHW> int run_fused(const Int8Args &a, int in, int out, hipStream_t s)
{
    if (out == DDCN_F32) launch_fused_of<DDCN_F32, NCHW>(a, in, s);
    else if (out == DDCN_BF16) launch_fused_of<DDCN_BF16, NCHW>(a, in, s);
    else launch_fused_of<DDCN_F16, NCHW>(a, in, s);
    return check_launch("int8 product");
}

Int8Args args_of(const ddcn_int8_geom *g)
{
    Int8Args a = {};
    a.plane = g->rows * g->cols;
    a.si = g->si; a.sh = g->sh; a.sw = g->sw; a.sk = g->sk;
    a.ldw = g->ldw;
    a.k = g->k; a.channels = g->channels; a.cols = g->cols; a.relu = g->relu;
    a.chunks = (int)ceil_div(g->k, 64) * 4;
    return a;
}

}  // namespace
}  // namespace ddcn

using namespace ddcn;

extern "C" {

size_t ddcn_int8_workspace_bytes(const ddcn_int8_geom *g)
{
    if (check(g, true) != DDCN_OK || !tokens_of(g)) return 0;
    const long long tokens = tokens_of(g);
    const long long pass = tokens < kPassTokens ? tokens : kPassTokens;
    const size_t aligned = plan_of(g, pass, true).bytes(), other = plan_of(g, pass, false).bytes();
    return aligned > other ? aligned : other;
}

int ddcn_int8_product(const void *x, const void *weight, const float *weight_scale, const float *bias, void *y,
                      void *workspace, size_t workspace_bytes, const ddcn_int8_geom *g, void *stream)
{
    int rc = check(g, true);
    if (rc != DDCN_OK) return rc;
    if (!tokens_of(g)) return DDCN_OK;
    const size_t need = ddcn_int8_workspace_bytes(g);
    if (!x || !weight || !weight_scale || !y || (need && !workspace)) return fail(DDCN_ERR_BAD_ARG, "a pointer is NULL");
    if ((uintptr_t)workspace & 255) return fail(DDCN_ERR_BAD_ARG, "workspace must be 256-byte aligned");
    if (workspace_bytes < need) return fail(DDCN_ERR_WORKSPACE, "workspace too small: %zu < %zu bytes", workspace_bytes, need);
    Int8Args a = args_of(g);
    a.x = x;
    a.w = (const signed char *)weight;
    a.w_scale = weight_scale;
    a.bias = bias;
    a.y = y;
    const long long total = tokens_of(g);
    for (a.t0 = 0; a.t0 < total; a.t0 += kPassTokens) {    // (later passes fit the first one's workspace)
        a.tokens = (int)(total - a.t0 < kPassTokens ? total - a.t0 : kPassTokens);
        const Plan p = plan_of(g, a.tokens, (((uintptr_t)weight | (uintptr_t)g->ldw) & 15) == 0 && g->ldw < (1LL << 25));
        if (p.how == kFused) {
            rc = g->nchw ? run_fused<true>(a, g->dtype, g->out_dtype, (hipStream_t)stream) : run_fused<false>(a, g->dtype, g->out_dtype, (hipStream_t)stream);
            if (rc != DDCN_OK) return rc;
            continue;
        }
        char *ws = (char *)workspace;
        a.ldq = a.tokens;
        a.q = (u32x4 *)ws;
        a.scale = (float *)(ws += p.q_bytes);
        a.wp = (u32x4 *)(ws += p.scale_bytes);
        a.part = (int *)(ws += p.w_bytes);
        a.splits = p.splits;
        a.steps_per = p.steps_per;
        if ((size_t)(ws - (char *)workspace) + p.part_bytes > workspace_bytes) return fail(DDCN_ERR_WORKSPACE, "workspace too small for the last pass");
        rc = run_prepare(a, g->dtype, p.how == kTiles, (hipStream_t)stream);
        if (rc != DDCN_OK) return rc;
        rc = g->nchw ? run_product<true>(a, p, g->out_dtype, (hipStream_t)stream) : run_product<false>(a, p, g->out_dtype, (hipStream_t)stream);
        if (rc != DDCN_OK) return rc;
    }
    return DDCN_OK;
}

int ddcn_int8_quantize(const void *x, void *q, long long ldq, float *scale, const ddcn_int8_geom *g, void *stream)
{
    int rc = check(g, false);
    if (rc != DDCN_OK) return rc;
    if (ldq < g->k) return fail(DDCN_ERR_SHAPE, "rows of %lld bytes hold no %d values", ldq, g->k);
    if (ldq > g->k + 64LL) return fail(DDCN_ERR_UNSUPPORTED, "rows of %lld bytes for %d values: at most 64 of padding", ldq, g->k);
    if (!tokens_of(g)) return DDCN_OK;
    if (!x || !q || !scale) return fail(DDCN_ERR_BAD_ARG, "a pointer is NULL");
    Int8Args a = args_of(g);
    a.x = x;
    a.q_rows = (signed char *)q;
    a.ldq = ldq;
    a.scale = scale;
    a.chunks = (int)ceil_div(ldq, 16);
    const long long total = tokens_of(g);
    for (a.t0 = 0; a.t0 < total; a.t0 += kPassTokens) {
        a.tokens = (int)(total - a.t0 < kPassTokens ? total - a.t0 : kPassTokens);
        rc = run_prepare(a, g->dtype, false, (hipStream_t)stream);
        if (rc != DDCN_OK) return rc;
    }
    return DDCN_OK;
}

}  // extern "C"
