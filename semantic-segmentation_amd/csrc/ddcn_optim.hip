// AdamW over many tensors in a few launches, moments in fp32 or in 8-bit codes, and the global gradient norm (gfx950).
// The formulas stand in include/ddcn_hip.h; they are evaluated here operation by operation, each rounded to fp32 (no
// fused multiply-adds in the moments), so that a code does not depend on how a compiler contracts an expression.
//
// The tensors of a launch travel as kernel arguments (up to 96 of them): no device table to keep, nothing that a later
// launch or another stream could overwrite.  One wave handles 256 consecutive elements of a tensor, four per lane -- in
// 8 bits a block of one pair of scales, whose maxima are one wave reduction.
#include <math.h>

#include "ddcn_elem.h"

namespace ddcn {
namespace {

constexpr int kBlock = 256;                     // elements per pair of scales, and per wave
constexpr int kWaves = 4;
constexpr int kBlocksPerWave = 4;
constexpr int kChunkBlocks = kWaves * kBlocksPerWave;   // blocks of a workgroup

struct AdamwTensor {
    void *p;
    const void *g;
    long long n;
    unsigned block0;       // first 256-element block in the arena
    unsigned chunk0;       // first workgroup of the launch
    float step_size;       // lr / (1 - beta1^t)
    float rsqrt_bc2;       // 1 / sqrt(1 - beta2^t)
};
constexpr int kMaxTensors = 96;
struct AdamwArgs {
    AdamwTensor t[kMaxTensors];
    void *m, *v;
    float *sm, *sv;
    const float *norm;
    float b1, ob1, b2, ob2, eps, decay, max_norm;
    unsigned seed;
    int count;
};
static_assert(sizeof(AdamwArgs) <= 4096, "kernel argument segment");

// The last entry whose first workgroup is not behind workgroup b
template <typename A>
__device__ __forceinline__ int find_tensor(const A &a, unsigned b)
{
    int lo = 0, hi = a.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.t[mid].chunk0 <= b) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Largest of non-negative floats over the wave, on their bits: ordered as the numbers are, NaN above infinity, so that
// one NaN is not lost
__device__ __forceinline__ unsigned wave_max_bits(unsigned x)
{
    for (int d = 32; d; d >>= 1) x = max(x, (unsigned)__shfl_xor((int)x, d));
    return x;
}

// Two 16-bit numbers for an element, from its place in the arena: multiply-xorshift with odd factors (first bits of the
// golden ratio and of the square roots of 17, 19, 2 and 11)
__device__ __forceinline__ unsigned noise(unsigned place, unsigned seed)
{
    unsigned h = place * 0x9E3779B1u + (seed * 0x1F83D9ABu + 0x5BE0CD19u);
    h = (h ^ (h >> 16)) * 0x6A09E667u;
    h = (h ^ (h >> 15)) * 0x510E527Fu;
    return h ^ (h >> 15);
}

constexpr unsigned kTiny = 0x0D800000u;      // 2^-100
constexpr unsigned kInf = 0x7F800000u;

// scale of a block with the largest value `bits`, and its reciprocal
__device__ __forceinline__ void block_scale(unsigned bits, float top2, float &scale, float &inverse)
{
#pragma clang fp contract(off)
    scale = bits < kTiny ? 0.f : bits >= kInf ? __uint_as_float(0x7FC00000u) : __uint_as_float(bits) / top2;
    inverse = bits < kTiny || bits >= kInf ? 0.f : 1.f / scale;
}

template <int DT, int BITS>
__global__ __launch_bounds__(64 * kWaves) void adamw_kernel(const AdamwArgs a)
{
#pragma clang fp contract(off)
    float c = 1.f;
    if (a.norm) {
        const float norm = *a.norm;
        if (!isfinite(norm)) return;
        c = fminf(1.f, a.max_norm / (norm + 1e-6f));
    }
    const int j = find_tensor(a, blockIdx.x);
    const AdamwTensor &t = a.t[j];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    constexpr unsigned kMask = DT == DDCN_F32 ? 15u : 7u;
    const bool vec_p = ((unsigned long long)t.p & kMask) == 0, vec_g = ((unsigned long long)t.g & kMask) == 0;
    const long long blocks = (t.n + kBlock - 1) / kBlock;
    for (int u = 0; u < kBlocksPerWave; ++u) {
        const long long blk = (long long)(blockIdx.x - t.chunk0) * kChunkBlocks + u * kWaves + wave;
        if (blk >= blocks) return;
        const long long i = blk * kBlock + lane * 4;                       // in the tensor
        const long long at = ((long long)t.block0 + blk) * kBlock + lane * 4;    // in the arena
        const int live = (int)min(max(t.n - i, 0LL), 4LL);
        float p[4], g[4], m[4], v[4], r[4];
        load_some<DT>(t.p, i, live, vec_p, p);
        load_some<DT>(t.g, i, live, vec_g, g);
        if (BITS == 32) {
            load_four<DDCN_F32>(a.m, at, m);
            load_four<DDCN_F32>(a.v, at, v);
        } else {
            const int qm = *(const int *)((const signed char *)a.m + at);
            const unsigned qv = *(const unsigned *)((const unsigned char *)a.v + at);
            const float sm = a.sm[t.block0 + blk], sv = a.sv[t.block0 + blk];
            for (int e = 0; e < 4; ++e) {
                const int q = (int)(signed char)(qm >> (8 * e)), w = (int)((qv >> (8 * e)) & 255u);
                m[e] = sm * (float)(q * abs(q));
                const float ro = sv * (float)(w * w);
                v[e] = ro * ro;
            }
        }
        unsigned top_m = 0, top_r = 0;
        for (int e = 0; e < 4; ++e) {
            const float ge = g[e] * c;
            m[e] = a.b1 * m[e] + a.ob1 * ge;
            v[e] = a.b2 * v[e] + (a.ob2 * ge) * ge;
            r[e] = sqrtf(v[e]);
            if (BITS == 8 && e >= live) m[e] = r[e] = 0.f;
            p[e] = p[e] * a.decay - t.step_size * (m[e] / (r[e] * t.rsqrt_bc2 + a.eps));
            top_m = max(top_m, __float_as_uint(fabsf(m[e])));
            top_r = max(top_r, __float_as_uint(fabsf(r[e])));
        }
        store_some<DT>(t.p, i, live, vec_p, p);
        if (BITS == 32) {
            // the arena is padded to whole blocks; what lies behind the tensor's end stays as it was
            store_some<DDCN_F32>(a.m, at, live, true, m);
            store_some<DDCN_F32>(a.v, at, live, true, v);
        } else {
            float sm, im, sv, iv;
            block_scale(wave_max_bits(top_m), 127.f * 127.f, sm, im);
            block_scale(wave_max_bits(top_r), 255.f * 255.f, sv, iv);
            unsigned qm = 0, qv = 0;
            for (int e = 0; e < 4; ++e) {
                const unsigned h = noise((unsigned)(at + e), a.seed);
                const float um = (float)(h & 0xFFFFu) * 0x1p-16f, uv = (float)(h >> 16) * 0x1p-16f;
                int q = im > 0.f ? (int)fminf(floorf(sqrtf(fabsf(m[e]) * im) + um), 127.f) : 0;
                if (m[e] < 0.f) q = -q;
                int w = iv > 0.f ? (int)fminf(floorf(sqrtf(r[e] * iv) + uv), 255.f) : 0;
                if (r[e] > 0.f && iv > 0.f) w = max(w, 1);
                qm |= (unsigned)(q & 255) << (8 * e);
                qv |= (unsigned)w << (8 * e);
            }
            *(unsigned *)((signed char *)a.m + at) = qm;
            *(unsigned *)((unsigned char *)a.v + at) = qv;
            if (lane == 0) {
                a.sm[t.block0 + blk] = sm;
                a.sv[t.block0 + blk] = sv;
            }
        }
    }
}

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
constexpr int kNormChunk = 16384;      // elements of a workgroup
struct NormTensor {
    const void *g;
    long long n;
    unsigned chunk0;
    int dtype;
};
constexpr int kMaxNorm = 160;
struct NormArgs {
    NormTensor t[kMaxNorm];
    double *partial;       // of this launch's first workgroup
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

template <int DT> __device__ __forceinline__ double chunk_square(const NormTensor &t, long long begin)
{
    constexpr unsigned kMask = DT == DDCN_F32 ? 15u : 7u;
    const bool vec = ((unsigned long long)t.g & kMask) == 0;
    const long long end = min(t.n, begin + kNormChunk);
    double s = 0.;
    for (long long i = begin + threadIdx.x * 4; i < end; i += 4 * 256) {
        float x[4];
        load_some<DT>(t.g, i, (int)min(end - i, 4LL), vec, x);
        for (int e = 0; e < 4; ++e) s += (double)x[e] * (double)x[e];
    }
    return s;
}

__global__ __launch_bounds__(256) void norm_partial_kernel(const NormArgs a)
{
    __shared__ double lds[4];
    const NormTensor &t = a.t[find_tensor(a, blockIdx.x)];
    const long long begin = (long long)(blockIdx.x - t.chunk0) * kNormChunk;
    double s = t.dtype == DDCN_F32 ? chunk_square<DDCN_F32>(t, begin)
               : t.dtype == DDCN_BF16 ? chunk_square<DDCN_BF16>(t, begin) : chunk_square<DDCN_F16>(t, begin);
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

template <int DT> void launch_adamw(int bits, unsigned grid, const AdamwArgs &a, hipStream_t s)
{
    if (bits == 32) adamw_kernel<DT, 32><<<grid, 64 * kWaves, 0, s>>>(a);
    else adamw_kernel<DT, 8><<<grid, 64 * kWaves, 0, s>>>(a);
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
        total += ceil_div(numels[i], kBlock) * kBlock;
    }
    if (total / kBlock >= (1LL << 32)) return fail(DDCN_ERR_UNSUPPORTED, "more than 2^40 elements in one arena");
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
    a.decay = (float)(1.0 - h->lr * h->weight_decay);
    a.max_norm = grad_norm ? (float)h->max_norm : 0.f;
    a.seed = h->seed;
    a.count = 0;
    long long chunks = 0, block = 0;
    int known = 0;
    float step_size = 0.f, rsqrt_bc2 = 0.f;
    for (int i = 0; i <= count; ++i) {
        const bool end = i == count;
        const long long blocks = end ? 0 : ceil_div(numels[i], kBlock), mine = ceil_div(blocks, kChunkBlocks);
        if (a.count && (end || a.count == kMaxTensors || chunks + mine >= (1LL << 31))) {
            const unsigned grid = (unsigned)chunks;
            hipStream_t s = (hipStream_t)stream;
            if (h->dtype == DDCN_F32) launch_adamw<DDCN_F32>(h->bits, grid, a, s);
            else if (h->dtype == DDCN_BF16) launch_adamw<DDCN_BF16>(h->bits, grid, a, s);
            else launch_adamw<DDCN_F16>(h->bits, grid, a, s);
            const int rc = check_launch("adamw");
            if (rc != DDCN_OK) return rc;
            a.count = 0;
            chunks = 0;
        }
        if (end) break;
        if (blocks && grads[i]) {
            if (mine >= (1LL << 31)) return fail(DDCN_ERR_UNSUPPORTED, "tensor %d has more than 2^43 elements", i);
            const int step = steps ? steps[i] : h->step;
            if (step != known) {
                step_size = (float)(h->lr / (1.0 - pow(h->beta1, step)));
                rsqrt_bc2 = (float)(1.0 / sqrt(1.0 - pow(h->beta2, step)));
                known = step;
            }
            AdamwTensor &t = a.t[a.count++];
            t.p = (void *)params[i];
            t.g = (const void *)grads[i];
            t.n = numels[i];
            t.block0 = (unsigned)block;
            t.chunk0 = (unsigned)chunks;
            t.step_size = step_size;
            t.rsqrt_bc2 = rsqrt_bc2;
            chunks += mine;
        }
        block += blocks;
    }
    return DDCN_OK;
}

int ddcn_adamw_moments(const void *exp_avg, const void *exp_avg_sq, const float *exp_avg_scale,
                       const float *exp_avg_sq_scale, float *m, float *v, long long numel, void *stream)
{
    if (numel < 0 || numel % kBlock) return fail(DDCN_ERR_SHAPE, "%lld elements: not a whole number of blocks of %d", numel, kBlock);
    if (!numel) return DDCN_OK;
    if (!exp_avg || !exp_avg_sq || !exp_avg_scale || !exp_avg_sq_scale || !m || !v) return fail(DDCN_ERR_BAD_ARG, "a pointer is NULL");
    if (((uintptr_t)m | (uintptr_t)v) & 15 || ((uintptr_t)exp_avg | (uintptr_t)exp_avg_sq) & 3)
        return fail(DDCN_ERR_BAD_ARG, "moments: outputs must be 16-byte, codes 4-byte aligned");
    const long long grid = ceil_div(numel / 4, 256);
    if (grid >= (1LL << 31)) return fail(DDCN_ERR_UNSUPPORTED, "%lld elements", numel);
    adamw_moments_kernel<<<(unsigned)grid, 256, 0, (hipStream_t)stream>>>((const signed char *)exp_avg,
        (const unsigned char *)exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, m, v, numel / 4);
    return check_launch("adamw_moments");
}

size_t ddcn_grad_norm_workspace_bytes(int count, const long long *numels)
{
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
        if (dtypes[i] < DDCN_F32 || dtypes[i] > DDCN_F16) return fail(DDCN_ERR_UNSUPPORTED, "dtype %d of tensor %d", dtypes[i], i);
        if (numels[i] && !grads[i]) return fail(DDCN_ERR_BAD_ARG, "tensor %d is NULL", i);
        if (grads[i] & (dtypes[i] == DDCN_F32 ? 3 : 1)) return fail(DDCN_ERR_BAD_ARG, "tensor %d is not aligned to its elements", i);
    }
    const size_t need = ddcn_grad_norm_workspace_bytes(count, numels);
    if (workspace_bytes < need) return fail(DDCN_ERR_WORKSPACE, "workspace too small: %zu < %zu bytes", workspace_bytes, need);
    NormArgs a;
    a.count = 0;
    long long chunks = 0, done = 0;
    for (int i = 0; i <= count; ++i) {
        const bool end = i == count;
        const long long mine = end ? 0 : ceil_div(numels[i], kNormChunk);
        if (a.count && (end || a.count == kMaxNorm || chunks + mine >= (1LL << 31))) {
            a.partial = (double *)workspace + done;
            norm_partial_kernel<<<(unsigned)chunks, 256, 0, (hipStream_t)stream>>>(a);
            const int rc = check_launch("grad_norm");
            if (rc != DDCN_OK) return rc;
            done += chunks;
            a.count = 0;
            chunks = 0;
        }
        if (end) break;
        if (!mine) continue;
        if (mine >= (1LL << 31)) return fail(DDCN_ERR_UNSUPPORTED, "tensor %d has %lld elements", i, numels[i]);
        NormTensor &t = a.t[a.count++];
        t.g = (const void *)grads[i];
        t.n = numels[i];
        t.chunk0 = (unsigned)chunks;
        t.dtype = dtypes[i];
        chunks += mine;
    }
    norm_final_kernel<<<1, 1024, 0, (hipStream_t)stream>>>((const double *)workspace, done, out);
    return check_launch("grad_norm");
}

}  // extern "C"
