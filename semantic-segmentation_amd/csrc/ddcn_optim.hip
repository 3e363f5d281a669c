// AdamW over many tensors in a few launches, moments in fp32 or in 8-bit codes, and the global gradient norm (gfx950).
// The formulas stand in include/ddcn_hip.h; they are evaluated here operation by operation, each rounded to fp32 (no
// fused multiply-adds in the moments), so that a code does not depend on how a compiler contracts an expression.
//
// The tensors of a launch travel as kernel arguments (up to 160 of them): no device table to keep, nothing that a later
// launch or another stream could overwrite.  One wave handles blocks of 256 consecutive elements of the arena, four per
// lane, whichever tensors they belong to -- in 8 bits a block is what one pair of scales stands for, and their maxima are
// one wave reduction.
#include <math.h>

#include "ddcn_elem.h"

namespace ddcn {
namespace {

constexpr int kBlock = 256;             // elements per pair of scales, and per wave and turn
constexpr int kWaves = 4;

constexpr long long kMaxGrid = 1LL << 23;   // workgroups of a launch: 256 threads each have to stay below 2^32 in all

constexpr int kMaxTensors = 160;
struct AdamwArgs {
    // tensor j of the launch covers the arena's blocks block0[j] .. block0[j+1]-1 (relative to `first`); n[j] elements.
    // A null gradient: blocks between the tensors that are left alone.
    void *p[kMaxTensors];
    const void *g[kMaxTensors];
    unsigned block0[kMaxTensors];
    unsigned n[kMaxTensors];
    void *m, *v;
    float *sm, *sv;
    const float *norm;
    long long first;       // block of the arena that the launch begins with
    unsigned blocks;       // of the launch
    float b1, ob1, b2, ob2, eps, max_norm;
    float decay, decay_rest;   // their sum is 1 - lr wd, to 48 bits
    float step_size;       // lr / (1 - beta1^t)
    float rsqrt_bc2;       // 1 / sqrt(1 - beta2^t)
    unsigned seed;
    int count;
};
static_assert(sizeof(AdamwArgs) <= 4096, "kernel argument segment");

// Largest of non-negative floats over the wave, on their bits: ordered as the numbers are, NaN above infinity, so that
// one NaN is not lost.  Five steps within and across rows of 16 lanes on the DPP network and one row broadcast; lane 63
// has the result.
__device__ __forceinline__ unsigned wave_max_bits(unsigned x)
{
#define DDCN_DPP_MAX(ctrl, rows) x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, rows, 0xf, false))
    DDCN_DPP_MAX(0x111, 0xf);       // row_shr:1
    DDCN_DPP_MAX(0x112, 0xf);       // row_shr:2
    DDCN_DPP_MAX(0x114, 0xf);       // row_shr:4
    DDCN_DPP_MAX(0x118, 0xf);       // row_shr:8
    DDCN_DPP_MAX(0x142, 0xa);       // row_bcast:15 into rows 1 and 3
    DDCN_DPP_MAX(0x143, 0xc);       // row_bcast:31 into rows 2 and 3
#undef DDCN_DPP_MAX
    return (unsigned)__builtin_amdgcn_readlane((int)x, 63);
}

// Two 16-bit numbers for an element, from its place in the arena: multiply-xorshift with odd factors (first bits of the
// golden ratio and of the square roots of 17, 19, 2 and 11).  `h`: place * golden + seed part
constexpr unsigned kGolden = 0x9E3779B1u;
__device__ __forceinline__ unsigned noise(unsigned h)
{
    h = (h ^ (h >> 16)) * 0x6A09E667u;
    h = (h ^ (h >> 15)) * 0x510E527Fu;
    return h ^ (h >> 15);
}

// Correctly rounded square root for x = 0 or x above 2^-96, where the hardware root (one unit off at most) needs no
// scaling: the neighbours' residuals decide.  Below, the result may be off by a unit of its own size (under 2^-48).
__device__ __forceinline__ float sqrt_rn(float x)
{
    float s = __builtin_amdgcn_sqrtf(x);
    const float dn = __uint_as_float(__float_as_uint(s) - 1u), up = __uint_as_float(__float_as_uint(s) + 1u);
    const float ed = fmaf(-dn, s, x), eu = fmaf(-up, s, x);
    s = ed <= 0.f ? dn : s;
    return eu > 0.f ? up : s;
}

constexpr unsigned kTiny = 0x0D800000u;      // 2^-100
constexpr unsigned kInf = 0x7F800000u;

struct Place {
    void *p;
    const void *g;
    long long i, at, block;    // element in the tensor (this lane's first), in the arena, block of the arena
    int live;                  // elements of this lane's four that exist
    bool wide;                 // all 256 elements exist and both addresses allow wide accesses
};

// What one lane holds of a block between its loads and its stores
template <int BITS> struct Held {
    float p[4], g[4], m[4], v[4];      // m, v: fp32 moments
    unsigned qm, qv;                   // or their codes and scales
    float sm, sv;
};

template <int DT, int BITS> __device__ __forceinline__ void load_block(const AdamwArgs &a, const Place &w, bool wide, Held<BITS> &h)
{
    if (wide) {
        load_four<DT>(w.p, w.i, h.p);
        load_four<DT>(w.g, w.i, h.g);
    } else {
        load_some<DT>(w.p, w.i, w.live, false, h.p);
        load_some<DT>(w.g, w.i, w.live, false, h.g);
    }
    if (BITS == 32) {
        load_four<DDCN_F32>(a.m, w.at, h.m);
        load_four<DDCN_F32>(a.v, w.at, h.v);
    } else {
        h.qm = *(const unsigned *)((const char *)a.m + w.at);
        h.qv = *(const unsigned *)((const char *)a.v + w.at);
        h.sm = a.sm[w.block];
        h.sv = a.sv[w.block];
    }
}

// The four codes of both moments.  EXACT: every root correctly rounded, as the codes are defined.  Otherwise from the
// hardware's roots: root + u is then off by less than 2^-15 (m: root <= 127, one unit of 2^-17 at the root and half a unit
// at the sum) and 2^-13 (r: root <= 255, relative 2^-21 from the root of v, the product with the reciprocal, the second
// root and the sum), so that its floor is the defined one unless it lies that close to a whole number -- `far` says how
// far the worst of them is from the middle between two.
template <bool EXACT>
__device__ __forceinline__ void encode(const float (&m)[4], const float (&v)[4], const float (&r)[4], float im, float iv,
                                       unsigned h0, unsigned &qm, unsigned &qv, float &far_m, float &far_r)
{
#pragma clang fp contract(off)
    qm = qv = 0;
    far_m = far_r = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const unsigned u = noise(h0 + (unsigned)e * kGolden);
        const float tm = fabsf(m[e]) * im, tr = (EXACT ? sqrtf(v[e]) : r[e]) * iv;
        // fma: the 16-bit number is exact, so that this is the one rounding of root + u
        const float xm = fmaf((float)(u & 0xFFFFu), 0x1p-16f, EXACT ? sqrt_rn(tm) : __builtin_amdgcn_sqrtf(tm));
        const float xr = fmaf((float)(u >> 16), 0x1p-16f, EXACT ? sqrt_rn(tr) : __builtin_amdgcn_sqrtf(tr));
        if (!EXACT) {
            far_m = fmaxf(far_m, fabsf(__builtin_amdgcn_fractf(xm) - 0.5f));
            far_r = fmaxf(far_r, fabsf(__builtin_amdgcn_fractf(xr) - 0.5f));
        }
        const int q = (int)copysignf(fminf(floorf(xm), 127.f), m[e]);
        qm |= (unsigned)(q & 255) << (8 * e);
        // at most 255, and at least 1 where v > 0
        qv = __builtin_amdgcn_cvt_pk_u8_f32(__builtin_amdgcn_fmed3f(floorf(xr), v[e] > 0.f ? 1.f : 0.f, 255.f), e, qv);
    }
}

// Lanes below 32 hold the largest |m| of a block, the others its largest r, as bits: their scales and reciprocals.
// x / 127^2 and x / 255^2 by the reciprocal and one residual, which is correctly rounded for these two divisors.
struct Scales {
    float sm, im, sv, iv;
};
__device__ __forceinline__ Scales block_scales(unsigned bits)
{
#pragma clang fp contract(off)
    const bool low = (threadIdx.x & 32) == 0;
    const float top2 = low ? 16129.f : 65025.f, rec = low ? 1.f / 16129.f : 1.f / 65025.f;
    const float x = __uint_as_float(bits), q0 = x * rec;
    const float s = fmaf(fmaf(-q0, top2, x), rec, q0);
    const float scale = bits < kTiny ? 0.f : bits >= kInf ? __uint_as_float(0x7FC00000u) : s;
    const float inverse = bits < kTiny || bits >= kInf ? 0.f : 1.f / s;
    auto lane = [](float f, int l) { return __uint_as_float((unsigned)__builtin_amdgcn_readlane((int)__float_as_uint(f), l)); };
    return Scales{lane(scale, 0), lane(inverse, 0), lane(scale, 32), lane(inverse, 32)};
}

template <int DT, int BITS>
__device__ __forceinline__ void update_block(const AdamwArgs &a, const Place &w, bool wide, float c, Held<BITS> &h)
{
#pragma clang fp contract(off)
    float m[4], v[4], r[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (BITS == 32) {
            m[e] = h.m[e];
            v[e] = h.v[e];
        } else {
            const float q = (float)(int)(signed char)(h.qm >> (8 * e)), k = (float)((h.qv >> (8 * e)) & 255u);
            m[e] = h.sm * (q * fabsf(q));                 // q|q| and k k are whole numbers below 2^24
            const float ro = h.sv * (k * k);
            v[e] = ro * ro;
        }
        const float ge = h.g[e] * c;
        m[e] = a.b1 * m[e] + a.ob1 * ge;
        v[e] = a.b2 * v[e] + (a.ob2 * ge) * ge;
        if (BITS == 8 && !wide && e >= w.live) m[e] = v[e] = 0.f;
    }
    // The parameter's own arithmetic may be fused and take the hardware's roots: nothing is decided on its last bits.
    // Without an eps that hides it, a root of the smallest numbers has to be right.
    // Small decays (lr wd below 2^-25 makes 1 - lr wd one in fp32) join the update before the one rounding at p.
    if (a.eps >= 0x1p-40f) {
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = __builtin_amdgcn_sqrtf(v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = sqrtf(v[e]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        h.p[e] = fmaf(h.p[e], a.decay, fmaf(-a.step_size, m[e] * __builtin_amdgcn_rcpf(fmaf(r[e], a.rsqrt_bc2, a.eps)), h.p[e] * a.decay_rest));
    if (wide) store_four<DT>(w.p, w.i, h.p);
    else store_some<DT>(w.p, w.i, w.live, false, h.p);
    if (BITS == 32) {
        // the arena is padded to whole blocks; what lies behind the tensor's end stays as it was
        if (wide) {
            store_four<DDCN_F32>(a.m, w.at, m);
            store_four<DDCN_F32>(a.v, w.at, v);
        } else {
            store_some<DDCN_F32>(a.m, w.at, w.live, true, m);
            store_some<DDCN_F32>(a.v, w.at, w.live, true, v);
        }
        return;
    }
    unsigned top_m = 0, top_v = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        top_m = max(top_m, __float_as_uint(m[e]) & 0x7FFFFFFFu);
        top_v = max(top_v, __float_as_uint(v[e]));         // never negative, nor -0
    }
    top_m = wave_max_bits(top_m);
    top_v = wave_max_bits(top_v) & 0x7FFFFFFFu;
    constexpr unsigned kSmall = 0x12800000u;               // 2^-90: below, the hardware's roots of v may be off
    const bool small = top_v < kSmall;
    const float top_r = small ? sqrtf(__uint_as_float(top_v)) : sqrt_rn(__uint_as_float(top_v));
    const Scales s = block_scales((threadIdx.x & 32) == 0 ? top_m : __float_as_uint(top_r));
    unsigned qm, qv;
    float far_m, far_r;
    const unsigned h0 = (unsigned)w.at * kGolden + (a.seed * 0x1F83D9ABu + 0x5BE0CD19u);
    encode<false>(m, v, r, s.im, s.iv, h0, qm, qv, far_m, far_r);
    if (small || __any(!(far_m < 0.5f - 0x1p-15f) || !(far_r < 0.5f - 0x1p-13f)))
        encode<true>(m, v, r, s.im, s.iv, h0, qm, qv, far_m, far_r);
    *(unsigned *)((char *)a.m + w.at) = qm;
    *(unsigned *)((char *)a.v + w.at) = qv;
    if ((threadIdx.x & 63) == 0) {
        a.sm[w.block] = s.sm;
        a.sv[w.block] = s.sv;
    }
}

// U blocks per wave, one after the other in the arena; where all of them are whole, every load is issued before the first
// result is needed.  Every byte moves once.  fp32 moments, 28 bytes an element: bound by HBM, 39.6 M elements in 185 us, 6.0
// TB/s.  8-bit ones, 16 bytes an element: 105 to 118 us for the same, 6.0 to 5.4 TB/s.  With bf16 parameters too, 10 bytes an
// element, its 100 VALU instructions -- decoding, hash, two roots and their rounding -- bound it: 45 M elements in 113 to 122 us,
// 4.0 TB/s.
template <int DT, int BITS, int U>
__global__ __launch_bounds__(64 * kWaves) void adamw_kernel(const AdamwArgs a)
{
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // the tensor of a block: how many of the sorted first blocks are not behind it, 64 compared at once
    unsigned b0[3];
    for (int i = 0; i < 3; ++i) b0[i] = lane + 64 * i < a.count ? a.block0[min(lane + 64 * i, kMaxTensors - 1)] : 0xFFFFFFFFu;
    float c = 1.f;
    if (a.norm) {
        const float norm = *a.norm;
        if (!isfinite(norm)) return;
        c = fminf(1.f, a.max_norm / (norm + 1e-6f));
    }
    constexpr unsigned kMask = DT == DDCN_F32 ? 15u : 7u;
    const unsigned first = (blockIdx.x * kWaves + wave) * U;
    auto place = [&](unsigned b) {
        Place w = {};
        if (b >= a.blocks) return w;
        int j = -1;
        for (int i = 0; i < 3; ++i) j += __popcll(__ballot(b0[i] <= b));
        w.p = a.p[j];
        w.g = a.g[j];
        const unsigned begin = (b - a.block0[j]) * kBlock, n = a.n[j];           // n at most 2^31
        w.i = (long long)begin + lane * 4;
        w.block = a.first + b;
        w.at = w.block * kBlock + lane * 4;
        w.live = (int)max(min((long long)n - w.i, 4LL), 0LL);
        w.wide = w.g && begin + kBlock <= n && (((unsigned long long)w.p | (unsigned long long)w.g) & kMask) == 0;
        return w;
    };
    Place w[U];
    bool all = true;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        w[u] = place(first + u);
        all = all && w[u].wide;
    }
    if (all) {
        Held<BITS> h[U];
#pragma unroll
        for (int u = 0; u < U; ++u) load_block<DT, BITS>(a, w[u], true, h[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) update_block<DT, BITS>(a, w[u], true, c, h[u]);
        return;
    }
#pragma unroll 1
    for (int u = 0; u < U; ++u) {
        const Place x = place(first + u);
        if (!x.g) continue;
        Held<BITS> h;
        load_block<DT, BITS>(a, x, x.wide, h);
        update_block<DT, BITS>(a, x, x.wide, c, h);
    }
}

// Bound by HBM: 2 bytes in and 8 out, 48 M elements in 75 us, 6.5 TB/s
__global__ __launch_bounds__(256) void adamw_moments_kernel(const signed char *m, const unsigned char *v, const float *sm,
                                                            const float *sv, float *om, float *ov, long long quads)
{
#pragma clang fp contract(off)
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= quads) return;
    const int qm = ((const int *)m)[i];
    const unsigned qv = ((const unsigned *)v)[i];
    const float a = sm[i / (kBlock / 4)], b = sv[i / (kBlock / 4)];
    f32x4 x, y;
    for (int e = 0; e < 4; ++e) {
        const int q = (int)(signed char)(qm >> (8 * e)), w = (int)((qv >> (8 * e)) & 255u);
        x[e] = a * (float)(q * abs(q));
        const float r = b * (float)(w * w);
        y[e] = r * r;
    }
    ((f32x4 *)om)[i] = x;
    ((f32x4 *)ov)[i] = y;
}

// ---------------------------------------------------------------- norm
constexpr int kNormChunk = 8192;       // elements of a workgroup
// 16 bytes a tensor, so that ResNet-50's 237 tensors fit one launch (62.6 us; two launches of 160 took 14.2 + 51.4 and a gap)
constexpr int kMaxNorm = 254;
constexpr unsigned kFirstChunk = 0x3FFFFFFFu;
struct NormArgs {
    const void *g[kMaxNorm];
    unsigned n[kMaxNorm];          // at most 2^31
    unsigned chunk0[kMaxNorm];     // first workgroup, and the element type in the two highest bits
    double *partial;               // of this launch's first workgroup
    int count;
};
static_assert(sizeof(NormArgs) <= 4096, "kernel argument segment");

__device__ __forceinline__ double block_sum(double s, double *lds)
{
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
    const int waves = blockDim.x >> 6;
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
    __syncthreads();
    s = 0.;
    for (int w = 0; w < waves; ++w) s += lds[w];
    return s;
}

template <int DT> __device__ __forceinline__ double chunk_square(const void *g, long long n, long long begin)
{
    constexpr unsigned kMask = DT == DDCN_F32 ? 15u : 7u;
    constexpr int kAhead = 8;          // wide loads in flight
    const bool vec = ((unsigned long long)g & kMask) == 0;
    const long long end = min(n, begin + kNormChunk);
    double s[4] = {0., 0., 0., 0.};
    if (vec && begin + kNormChunk <= n) {
#pragma unroll
        for (int k = 0; k < kNormChunk / 1024; k += kAhead) {
            float x[kAhead][4];
#pragma unroll
            for (int l = 0; l < kAhead; ++l) load_four<DT>(g, begin + (k + l) * 1024 + threadIdx.x * 4, x[l]);
#pragma unroll
            for (int l = 0; l < kAhead; ++l)
                for (int e = 0; e < 4; ++e) s[e] = fma((double)x[l][e], (double)x[l][e], s[e]);
        }
    } else {
        for (long long i = begin + threadIdx.x * 4; i < end; i += 1024) {
            float x[4];
            load_some<DT>(g, i, (int)min(end - i, 4LL), vec, x);
            for (int e = 0; e < 4; ++e) s[e] = fma((double)x[e], (double)x[e], s[e]);
        }
    }
    return (s[0] + s[1]) + (s[2] + s[3]);
}

// Sums in fp64 (the adds hide behind the loads), a workgroup a chunk, their sums in a fixed order by one workgroup: no
// atomics.  Read-only: 48 M fp32 elements in 42 us where they come from HBM alone, 62 right after a step, whose writes
// are then still leaving the last-level cache.
__global__ __launch_bounds__(256) void norm_partial_kernel(const NormArgs a)
{
    __shared__ double lds[4];
    // the last tensor whose first workgroup is not behind this one, 64 compared at once
    const int lane = threadIdx.x & 63;
    int j = -1;
    for (int i = 0; i < 4; ++i) {
        const unsigned c0 = lane + 64 * i < a.count ? a.chunk0[min(lane + 64 * i, kMaxNorm - 1)] & kFirstChunk : 0xFFFFFFFFu;
        j += __popcll(__ballot(c0 <= blockIdx.x));
    }
    const void *g = a.g[j];
    const unsigned dtype = a.chunk0[j] >> 30;
    const long long n = a.n[j], begin = (long long)(blockIdx.x - (a.chunk0[j] & kFirstChunk)) * kNormChunk;
    double s = dtype == DDCN_F32 ? chunk_square<DDCN_F32>(g, n, begin)
               : dtype == DDCN_BF16 ? chunk_square<DDCN_BF16>(g, n, begin) : chunk_square<DDCN_F16>(g, n, begin);
    s = block_sum(s, lds);
    if (threadIdx.x == 0) a.partial[blockIdx.x] = s;
}

__global__ __launch_bounds__(1024) void norm_final_kernel(const double *partial, long long n, float *out)
{
    __shared__ double lds[16];
    double s = 0.;
    for (long long i = threadIdx.x; i < n; i += 1024) s += partial[i];
    s = block_sum(s, lds);
    if (threadIdx.x == 0) *out = (float)sqrt(s);
}

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// Blocks per wave.  fp32 moments: one (the large launch of ResNet-50's 41 M parameters takes 185 us, 190 with two or four).
// 8 bits: two, whose loads then hide behind the other's arithmetic (107 us; 123 with one, 110 with four, in turn) -- but one where
// two would leave CUs without work.
constexpr unsigned kSpreadBlocks = 8192;
// Blocks of tensors without a gradient that a launch may hold between two others, as one entry whose waves end at once: below,
// they cost less than a launch more (two tensors of 16 blocks, fp32: 4.5 us in two launches; in one 2.6 with 1024 blocks
// between them, 3.6 with 8192, 4.8 with 16384, 42 with 262144; with 8-bit moments 6.1, and 3.4, 5.7, 7.0, 48).
constexpr long long kMaxGap = 8192;
template <int DT, int BITS> void launch_adamw(const AdamwArgs &a, hipStream_t s)
{
    constexpr int kMany = BITS == 32 ? 1 : 2;
    if (kMany == 1 || a.blocks <= kSpreadBlocks)
        adamw_kernel<DT, BITS, 1><<<(unsigned)ceil_div(a.blocks, kWaves), 64 * kWaves, 0, s>>>(a);
    else
        adamw_kernel<DT, BITS, kMany><<<(unsigned)ceil_div(a.blocks, kMany * kWaves), 64 * kWaves, 0, s>>>(a);
}

}  // namespace
}  // namespace ddcn

using namespace ddcn;

extern "C" {

long long ddcn_adamw_arena(int count, const long long *numels)
{
    if (count < 0 || (count && !numels)) return fail(DDCN_ERR_BAD_ARG, "ddcn_adamw_arena: count %d", count);
    long long total = 0;
    for (int i = 0; i < count; ++i) {
        if (numels[i] < 0 || numels[i] > (1LL << 40)) return fail(DDCN_ERR_SHAPE, "tensor %d has %lld elements", i, numels[i]);
        total += ceil_div(numels[i], kBlock) * kBlock;         // (stays below 2^42)
        if (total / kBlock >= (1LL << 32)) return fail(DDCN_ERR_UNSUPPORTED, "more than 2^40 elements in one arena");
    }
    return total;
}

int ddcn_adamw_step(int count, const unsigned long long *params, const unsigned long long *grads,
                    const long long *numels, const int *steps, void *exp_avg, void *exp_avg_sq, float *exp_avg_scale,
                    float *exp_avg_sq_scale, const float *grad_norm, const ddcn_adamw_hyper *h, void *stream)
{
    if (!h) return fail(DDCN_ERR_BAD_ARG, "hyper is NULL");
    const long long arena = ddcn_adamw_arena(count, numels);
    if (arena < 0) return (int)arena;
    if (!arena) return DDCN_OK;
    if (!params || !grads || !exp_avg || !exp_avg_sq) return fail(DDCN_ERR_BAD_ARG, "a pointer is NULL");
    if (h->bits != 32 && h->bits != 8) return fail(DDCN_ERR_UNSUPPORTED, "moments of %d bits (32 or 8)", h->bits);
    if (h->bits == 8 && (!exp_avg_scale || !exp_avg_sq_scale)) return fail(DDCN_ERR_BAD_ARG, "8-bit moments need their scales");
    if (h->dtype < DDCN_F32 || h->dtype > DDCN_F16) return fail(DDCN_ERR_UNSUPPORTED, "dtype %d", h->dtype);
    if (((uintptr_t)exp_avg | (uintptr_t)exp_avg_sq) & 15) return fail(DDCN_ERR_BAD_ARG, "the arena must be 16-byte aligned");
    if (!(h->lr >= 0) || !(h->beta1 >= 0 && h->beta1 < 1) || !(h->beta2 >= 0 && h->beta2 < 1) || !(h->eps >= 0) ||
        !(h->weight_decay >= 0) || (grad_norm && !(h->max_norm > 0)))
        return fail(DDCN_ERR_BAD_ARG, "lr %g beta1 %g beta2 %g eps %g weight_decay %g max_norm %g", h->lr, h->beta1, h->beta2,
                    h->eps, h->weight_decay, h->max_norm);
    const unsigned size = h->dtype == DDCN_F32 ? 4 : 2;
    for (int i = 0; i < count; ++i) {
        if (numels[i] && grads[i] && !params[i]) return fail(DDCN_ERR_BAD_ARG, "tensor %d is NULL", i);
        if ((params[i] | grads[i]) & (size - 1)) return fail(DDCN_ERR_BAD_ARG, "tensor %d is not aligned to its elements", i);
        if ((steps ? steps[i] : h->step) < 1) return fail(DDCN_ERR_BAD_ARG, "step of tensor %d is below 1", i);
    }
    AdamwArgs a;
    a.m = exp_avg;
    a.v = exp_avg_sq;
    a.sm = exp_avg_scale;
    a.sv = exp_avg_sq_scale;
    a.norm = grad_norm;
    a.b1 = (float)h->beta1;
    a.ob1 = (float)(1.0 - h->beta1);
    a.b2 = (float)h->beta2;
    a.ob2 = (float)(1.0 - h->beta2);
    a.eps = (float)h->eps;
    // 1 - lr wd towards zero, and the rest, of the same sign and never zero beside it: an infinite p stays infinite
    const double decay = 1.0 - h->lr * h->weight_decay;
    a.decay = (float)decay;
    if (fabs((double)a.decay) > fabs(decay)) a.decay = nextafterf(a.decay, 0.f);
    a.decay_rest = a.decay == 0.f ? 0.f : (float)copysign(fmax(fabs(decay - a.decay), 0x1p-100), decay);
    a.max_norm = grad_norm ? (float)h->max_norm : 0.f;
    a.seed = h->seed;
    a.count = 0;
    a.blocks = 0;
    a.first = 0;
    a.step_size = a.rsqrt_bc2 = 0.f;
    long long block = 0;       // of the arena, where the next tensor starts
    int known = 0;
    auto launch = [&]() -> int {
        const bool due = a.count > 0;
        if (due) {
            hipStream_t s = (hipStream_t)stream;
            if (h->dtype == DDCN_F32) h->bits == 32 ? launch_adamw<DDCN_F32, 32>(a, s) : launch_adamw<DDCN_F32, 8>(a, s);
            else if (h->dtype == DDCN_BF16) h->bits == 32 ? launch_adamw<DDCN_BF16, 32>(a, s) : launch_adamw<DDCN_BF16, 8>(a, s);
            else h->bits == 32 ? launch_adamw<DDCN_F16, 32>(a, s) : launch_adamw<DDCN_F16, 8>(a, s);
        }
        a.count = 0;
        a.blocks = 0;
        return due ? check_launch("adamw") : DDCN_OK;
    };
    for (int i = 0; i < count; ++i) {
        if (!grads[i] || !numels[i]) {        // no gradient: its step number does not matter either
            block += ceil_div(numels[i], kBlock);
            continue;
        }
        const int step = steps ? steps[i] : h->step;
        if (step != known) {       // one step number to a launch
            const int rc = launch();
            if (rc != DDCN_OK) return rc;
            a.step_size = (float)(h->lr / (1.0 - pow(h->beta1, step)));
            a.rsqrt_bc2 = (float)(1.0 / sqrt(1.0 - pow(h->beta2, step)));
            known = step;
        }
        // a tensor of 2^31 elements and more goes in pieces
        for (long long done = 0; done < numels[i]; done += 1LL << 31) {
            const long long n = numels[i] - done < (1LL << 31) ? numels[i] - done : 1LL << 31, blocks = ceil_div(n, kBlock);
            // blocks of the arena since the launch's last tensor, of tensors without a gradient
            const long long gap = a.count ? block - (a.first + a.blocks) : 0;
            if (gap > kMaxGap || a.count + (gap > 0) >= kMaxTensors || a.blocks + gap + blocks > kMaxGrid * kWaves) {
                const int rc = launch();
                if (rc != DDCN_OK) return rc;
            }
            if (!a.count) a.first = block;
            else if (gap) {
                a.p[a.count] = nullptr;
                a.g[a.count] = nullptr;
                a.block0[a.count] = a.blocks;
                a.n[a.count++] = 0;
                a.blocks += (unsigned)gap;
            }
            a.p[a.count] = (void *)(params[i] + done * size);
            a.g[a.count] = (const void *)(grads[i] + done * size);
            a.block0[a.count] = a.blocks;
            a.n[a.count++] = (unsigned)n;
            a.blocks += (unsigned)blocks;
            block += blocks;
        }
    }
    return launch();
}

int ddcn_adamw_moments(const void *exp_avg, const void *exp_avg_sq, const float *exp_avg_scale,
                       const float *exp_avg_sq_scale, float *m, float *v, long long numel, void *stream)
{
    if (numel < 0 || numel % kBlock) return fail(DDCN_ERR_SHAPE, "%lld elements: not a whole number of blocks of %d", numel, kBlock);
    if (!numel) return DDCN_OK;
    if (!exp_avg || !exp_avg_sq || !exp_avg_scale || !exp_avg_sq_scale || !m || !v) return fail(DDCN_ERR_BAD_ARG, "a pointer is NULL");
    if (((uintptr_t)m | (uintptr_t)v) & 15 || ((uintptr_t)exp_avg | (uintptr_t)exp_avg_sq) & 3)
        return fail(DDCN_ERR_BAD_ARG, "moments: outputs must be 16-byte, codes 4-byte aligned");
    for (long long at = 0; at < numel; at += kMaxGrid * 1024) {
        const long long quads = (numel - at < kMaxGrid * 1024 ? numel - at : kMaxGrid * 1024) / 4;
        adamw_moments_kernel<<<(unsigned)ceil_div(quads, 256), 256, 0, (hipStream_t)stream>>>((const signed char *)exp_avg + at,
            (const unsigned char *)exp_avg_sq + at, exp_avg_scale + at / kBlock, exp_avg_sq_scale + at / kBlock, m + at, v + at, quads);
        const int rc = check_launch("adamw_moments");
        if (rc != DDCN_OK) return rc;
    }
    return DDCN_OK;
}

size_t ddcn_grad_norm_workspace_bytes(int count, const long long *numels)
{
    if (count < 0 || (count && !numels)) return 0;
    long long chunks = 0;
    for (int i = 0; i < count; ++i) chunks += ceil_div(numels[i] > 0 ? numels[i] : 0, kNormChunk);
    return round_up((size_t)(chunks > 0 ? chunks : 1) * sizeof(double), 256);
}

int ddcn_grad_norm(int count, const unsigned long long *grads, const long long *numels, const int *dtypes, float *out,
                   void *workspace, size_t workspace_bytes, void *stream)
{
    if (count < 0 || (count && (!grads || !numels || !dtypes)) || !out || !workspace) return fail(DDCN_ERR_BAD_ARG, "a pointer is NULL");
    if ((uintptr_t)workspace & 15) return fail(DDCN_ERR_BAD_ARG, "workspace must be 16-byte aligned");
    for (int i = 0; i < count; ++i) {
        if (numels[i] < 0) return fail(DDCN_ERR_SHAPE, "tensor %d has %lld elements", i, numels[i]);
        if (numels[i] > kMaxGrid * kNormChunk) return fail(DDCN_ERR_UNSUPPORTED, "tensor %d has %lld elements", i, numels[i]);
        if (dtypes[i] < DDCN_F32 || dtypes[i] > DDCN_F16) return fail(DDCN_ERR_UNSUPPORTED, "dtype %d of tensor %d", dtypes[i], i);
        if (numels[i] && !grads[i]) return fail(DDCN_ERR_BAD_ARG, "tensor %d is NULL", i);
        if (grads[i] & (dtypes[i] == DDCN_F32 ? 3 : 1)) return fail(DDCN_ERR_BAD_ARG, "tensor %d is not aligned to its elements", i);
    }
    const size_t need = ddcn_grad_norm_workspace_bytes(count, numels);
    if (workspace_bytes < need) return fail(DDCN_ERR_WORKSPACE, "workspace too small: %zu < %zu bytes", workspace_bytes, need);
    NormArgs a;
    a.count = 0;
    long long chunks = 0, done = 0;
    auto launch = [&]() -> int {
        if (!a.count) return DDCN_OK;
        a.partial = (double *)workspace + done;
        norm_partial_kernel<<<(unsigned)chunks, 256, 0, (hipStream_t)stream>>>(a);
        done += chunks;
        a.count = 0;
        chunks = 0;
        return check_launch("grad_norm");
    };
    for (int i = 0; i < count; ++i)
        for (long long at = 0; at < numels[i]; at += 1LL << 31) {      // (whole chunks)
            const long long n = numels[i] - at < (1LL << 31) ? numels[i] - at : 1LL << 31, mine = ceil_div(n, kNormChunk);
            if (a.count == kMaxNorm || chunks + mine > kMaxGrid) {
                const int rc = launch();
                if (rc != DDCN_OK) return rc;
            }
            a.g[a.count] = (const void *)(grads[i] + at * (dtypes[i] == DDCN_F32 ? 4 : 2));
            a.n[a.count] = (unsigned)n;
            a.chunk0[a.count++] = (unsigned)chunks | (unsigned)dtypes[i] << 30;
            chunks += mine;
        }
    const int rc = launch();
    if (rc != DDCN_OK) return rc;
    norm_final_kernel<<<1, 1024, 0, (hipStream_t)stream>>>((const double *)workspace, done, out);
    return check_launch("grad_norm");
}

}  // extern "C"
