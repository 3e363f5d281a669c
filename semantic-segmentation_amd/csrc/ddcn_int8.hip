// Linear layers and 1x1 convolutions in 8-bit integers, a scale per token and per output channel (gfx950).  The formulas
// stand in include/ddcn_hip.h.
//
//   quantize_rows / quantize_map   x (any strides) -> q int8 [token][ldq], zero from k to ldq, and the tokens' scales
//   product                        q x weight^T on v_mfma_i32_16x16x64_i8, exact int32 sums, scales + bias + ReLU in the
//                                  epilogue
#include "ddcn_elem.h"

namespace ddcn {
namespace {

typedef __attribute__((ext_vector_type(4))) int i32x4;

constexpr int kPadK = 128;             // rows of q are padded to this many bytes
constexpr int kMaxK = 131072;          // k * 127 * 128 stays below 2^31

struct Int8Args {
    const void *x;
    signed char *q;
    float *scale;
    const signed char *w;
    const float *w_scale, *bias;
    void *y;
    long long tokens, plane;           // plane = rows * cols
    long long si, sh, sw, sk, ldq, ldw;
    int k, channels, cols, relu;
};

// first element of token t in x
__device__ __forceinline__ long long token_base(const Int8Args &a, long long t)
{
    const long long img = t / a.plane, p = t - img * a.plane;
    const long long h = p / a.cols;
    return img * a.si + h * a.sh + (p - h * a.cols) * a.sw;
}

// Scale and factor from the largest |x| of a token, given as its bits (ordered as the numbers are, NaN on top)
__device__ __forceinline__ void token_scale(unsigned top, float &scale, float &factor)
{
    constexpr unsigned kLeast = 0x0F800000u, kInf = 0x7F800000u;      // 2^-96
    if (top >= kInf) {
        scale = __uint_as_float(0x7FC00000u);
        factor = 0.f;
        return;
    }
    const float m = __uint_as_float(max(top, kLeast));
    scale = m / 127.f;
    factor = 127.f / m;
}
// one code; factor 0 marks a token with a NaN or an infinity: its codes are 0 and its scale is NaN
__device__ __forceinline__ unsigned code(float x, float factor)
{
    return factor > 0.f ? (unsigned)(int)rintf(x * factor) & 255u : 0u;
}

// sk == 1: a wave per token
template <int DT> __global__ __launch_bounds__(256) void quantize_rows_kernel(const Int8Args a)
{
    const int lane = threadIdx.x & 63;
    const long long t = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= a.tokens) return;
    const long long base = token_base(a, t);
    unsigned top = 0;
    for (int k = lane; k < a.k; k += 64) top = max(top, __float_as_uint(fabsf(load_one<DT>(a.x, base + k))));
    for (int d = 32; d; d >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, d));
    float scale, factor;
    token_scale(top, scale, factor);
    signed char *q = a.q + t * a.ldq;
    for (long long k = lane; k < a.ldq; k += 64) q[k] = k < a.k ? (signed char)code(load_one<DT>(a.x, base + k), factor) : 0;
    if (lane == 0) a.scale[t] = scale;
}

// any strides, lanes along the tokens: 64 tokens per workgroup, the channels dealt to its four waves
template <int DT> __global__ __launch_bounds__(256) void quantize_map_kernel(const Int8Args a)
{
    __shared__ unsigned tops[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long t = (long long)blockIdx.x * 64 + lane;
    const bool live = t < a.tokens;
    const long long base = live ? token_base(a, t) : 0;
    unsigned top = 0;
    if (live)
        for (int k = wave; k < a.k; k += 4) top = max(top, __float_as_uint(fabsf(load_one<DT>(a.x, base + k * a.sk))));
    tops[wave][lane] = top;
    __syncthreads();
    top = max(max(tops[0][lane], tops[1][lane]), max(tops[2][lane], tops[3][lane]));
    if (!live) return;
    float scale, factor;
    token_scale(top, scale, factor);
    signed char *q = a.q + t * a.ldq;
    for (long long k = wave; k < a.ldq; k += 4)
        q[k] = k < a.k ? (signed char)code(load_one<DT>(a.x, base + k * a.sk), factor) : 0;
    if (wave == 0) a.scale[t] = scale;
}

// 16 weight bytes from k on, zero behind the row's k bytes
__device__ __forceinline__ i32x4 weight_chunk(const signed char *row, int k, int kk, bool wide)
{
    if (wide && k + 16 <= kk) return *(const i32x4 *)(row + k);
    union {
        signed char b[16];
        i32x4 v;
    } u;
    for (int e = 0; e < 16; ++e) u.b[e] = k + e < kk ? row[k + e] : 0;
    return u.v;
}

// 64 x 64 per workgroup, 32 x 32 per wave.  The operand whose index runs along the lanes of the result is the one that is
// contiguous in y: tokens for nchw, channels otherwise.
template <int DT, bool NCHW> __global__ __launch_bounds__(256) void product_kernel(const Int8Args a)
{
#pragma clang fp contract(off)
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long t0 = (long long)blockIdx.x * 64 + (wave & 1) * 32;
    const int n0 = blockIdx.y * 64 + (wave >> 1) * 32;
    const int r16 = lane & 15, kc = (lane >> 4) * 16;
    const bool wide = (((unsigned long long)a.w | (unsigned long long)a.ldw) & 15) == 0;
    i32x4 acc[2][2] = {};
    const i32x4 zero = {0, 0, 0, 0};
    for (int k0 = 0; k0 < a.k; k0 += 64) {
        i32x4 ft[2], fw[2];
        for (int i = 0; i < 2; ++i) {
            const long long t = t0 + i * 16 + r16;
            const int n = n0 + i * 16 + r16;
            ft[i] = t < a.tokens ? *(const i32x4 *)(a.q + t * a.ldq + k0 + kc) : zero;
            fw[i] = n < a.channels ? weight_chunk(a.w + n * a.ldw, k0 + kc, a.k, wide) : zero;
        }
        for (int i = 0; i < 2; ++i)
            for (int j = 0; j < 2; ++j)
                acc[i][j] = NCHW ? __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[i], ft[j], acc[i][j], 0, 0, 0)
                                 : __builtin_amdgcn_mfma_i32_16x16x64_i8(ft[i], fw[j], acc[i][j], 0, 0, 0);
    }
    // lane l holds rows 4 * (l / 16) + e, column l % 16 of each 16 x 16 tile
    for (int i = 0; i < 2; ++i)
        for (int j = 0; j < 2; ++j)
            for (int e = 0; e < 4; ++e) {
                const int along = j * 16 + r16, across = i * 16 + (lane >> 4) * 4 + e;
                const long long t = t0 + (NCHW ? along : across);
                const int n = n0 + (NCHW ? across : along);
                if (t >= a.tokens || n >= a.channels) continue;
                float v = (float)acc[i][j][e] * (a.scale[t] * a.w_scale[n]);
                if (a.bias) v = v + a.bias[n];
                if (a.relu && v < 0.f) v = 0.f;
                const long long img = t / a.plane;
                const long long at = NCHW ? (img * a.channels + n) * a.plane + (t - img * a.plane) : t * a.channels + n;
                store_one<DT>(a.y, at, v);
            }
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
size_t q_bytes(const ddcn_int8_geom *g) { return round_up((size_t)tokens_of(g) * round_up(g->k, kPadK), 256); }

int run_quantize(const Int8Args &a, int dtype, hipStream_t s)
{
    if (a.sk == 1) {
        const unsigned grid = (unsigned)ceil_div(a.tokens, 4);
        if (dtype == DDCN_F32) quantize_rows_kernel<DDCN_F32><<<grid, 256, 0, s>>>(a);
        else if (dtype == DDCN_BF16) quantize_rows_kernel<DDCN_BF16><<<grid, 256, 0, s>>>(a);
        else quantize_rows_kernel<DDCN_F16><<<grid, 256, 0, s>>>(a);
    } else {
        const unsigned grid = (unsigned)ceil_div(a.tokens, 64);
        if (dtype == DDCN_F32) quantize_map_kernel<DDCN_F32><<<grid, 256, 0, s>>>(a);
        else if (dtype == DDCN_BF16) quantize_map_kernel<DDCN_BF16><<<grid, 256, 0, s>>>(a);
        else quantize_map_kernel<DDCN_F16><<<grid, 256, 0, s>>>(a);
    }
    return check_launch("int8 quantize");
}

template <bool NCHW> void run_product(const Int8Args &a, int dtype, hipStream_t s)
{
    const dim3 grid((unsigned)ceil_div(a.tokens, 64), (unsigned)ceil_div(a.channels, 64));
    if (dtype == DDCN_F32) product_kernel<DDCN_F32, NCHW><<<grid, 256, 0, s>>>(a);
    else if (dtype == DDCN_BF16) product_kernel<DDCN_BF16, NCHW><<<grid, 256, 0, s>>>(a);
    else product_kernel<DDCN_F16, NCHW><<<grid, 256, 0, s>>>(a);
}

Int8Args args_of(const ddcn_int8_geom *g)
{
    Int8Args a = {};
    a.tokens = tokens_of(g);
    a.plane = (long long)g->rows * g->cols;
    a.si = g->si; a.sh = g->sh; a.sw = g->sw; a.sk = g->sk;
    a.ldw = g->ldw;
    a.k = g->k; a.channels = g->channels; a.cols = g->cols; a.relu = g->relu;
    return a;
}

}  // namespace
}  // namespace ddcn

using namespace ddcn;

extern "C" {

size_t ddcn_int8_workspace_bytes(const ddcn_int8_geom *g)
{
    if (check(g, false) != DDCN_OK) return 0;
    return q_bytes(g) + round_up((size_t)tokens_of(g) * sizeof(float), 256);
}

int ddcn_int8_product(const void *x, const void *weight, const float *weight_scale, const float *bias, void *y,
                      void *workspace, size_t workspace_bytes, const ddcn_int8_geom *g, void *stream)
{
    int rc = check(g, true);
    if (rc != DDCN_OK) return rc;
    if (!tokens_of(g)) return DDCN_OK;
    if (!x || !weight || !weight_scale || !y || !workspace) return fail(DDCN_ERR_BAD_ARG, "a pointer is NULL");
    if ((uintptr_t)workspace & 255) return fail(DDCN_ERR_BAD_ARG, "workspace must be 256-byte aligned");
    const size_t need = ddcn_int8_workspace_bytes(g);
    if (workspace_bytes < need) return fail(DDCN_ERR_WORKSPACE, "workspace too small: %zu < %zu bytes", workspace_bytes, need);
    Int8Args a = args_of(g);
    a.x = x;
    a.q = (signed char *)workspace;
    a.scale = (float *)((char *)workspace + q_bytes(g));
    a.ldq = (long long)round_up(g->k, kPadK);
    a.w = (const signed char *)weight;
    a.w_scale = weight_scale;
    a.bias = bias;
    a.y = y;
    rc = run_quantize(a, g->dtype, (hipStream_t)stream);
    if (rc != DDCN_OK) return rc;
    if (g->nchw) run_product<true>(a, g->out_dtype, (hipStream_t)stream);
    else run_product<false>(a, g->out_dtype, (hipStream_t)stream);
    return check_launch("int8 product");
}

int ddcn_int8_quantize(const void *x, void *q, long long ldq, float *scale, const ddcn_int8_geom *g, void *stream)
{
    const int rc = check(g, false);
    if (rc != DDCN_OK) return rc;
    if (ldq < g->k) return fail(DDCN_ERR_SHAPE, "rows of %lld bytes hold no %d values", ldq, g->k);
    if (!tokens_of(g)) return DDCN_OK;
    if (!x || !q || !scale) return fail(DDCN_ERR_BAD_ARG, "a pointer is NULL");
    Int8Args a = args_of(g);
    a.x = x;
    a.q = (signed char *)q;
    a.ldq = ldq;
    a.scale = scale;
    return run_quantize(a, g->dtype, (hipStream_t)stream);
}

}  // extern "C"
