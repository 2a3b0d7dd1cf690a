// mx.cu -- microscaled matrices: tcg_mx_quantize, tcg_mx_dequantize, and the residual's addition with the
// root-mean-square norm whose rows come out in 8 or 4 bits (tcg_add_rms_norm).
//
// A block of 32 columns has the scale 2^s, s = floor(log2 max|x|) - m, m = 2 for E2M1 (largest value 6 = 1.5 * 2^2) and 8
// for E4M3 (448 = 1.75 * 2^8), and codes rn(x / 2^s). floor(log2) is the exponent field of the largest magnitude, and the
// division by a power of two is exact, so codes are the format's nearest values to the inputs themselves.
//
// The norm's codes have to be those of y = h / sqrt(mean(h^2) + eps) * w, not of an fp32 approximation that may lie on
// the other side of the border between two codes. The sum of squares and the root are taken in 64 bits; the products in
// two fp32 numbers (y + rest, good to 2^-46), and before y is rounded to fewer bits its last bit is made odd where a rest
// is left: a rounding to odd, after which the second rounding cannot meet a tie that is none. That is ~12 fp32 operations
// a value instead of 64-bit conversions, whose rate (16 a cycle and SM) is half of what the memory delivers for 16-bit rows.
#include "mx.cuh"

#include <cuda_fp4.h>
#include <cuda_fp8.h>

namespace tcg {
namespace {

constexpr int LANE = 8;             // consecutive columns of a lane: 4 lanes make a block, 16 a word of scales
constexpr int MX_WARPS = 8;

// 8 elements from p, of which `left` exist (the rest are 0); `vec`: p is 16-byte aligned where all 8 exist.
template <typename T>
__device__ __forceinline__ void load8(const T *p, long long left, bool vec, float (&x)[LANE])
{
    if (vec && left >= LANE) {
        constexpr int V = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < LANE; i += V) {
            float k[V];
            load_pack<T, V>(p + i, k);
#pragma unroll
            for (int j = 0; j < V; j++) x[i + j] = k[j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < LANE; i++) x[i] = i < left ? to_f32(p[i]) : 0.0f;
    }
}
template <typename T>
__device__ __forceinline__ void store8(T *p, long long left, bool vec, const float (&x)[LANE])
{
    if (vec && left >= LANE) {
        constexpr int V = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < LANE; i += V) {
            float k[V];
#pragma unroll
            for (int j = 0; j < V; j++) k[j] = x[i + j];
            store_pack<T, V>(p + i, k);
        }
    } else {
#pragma unroll
        for (int i = 0; i < LANE; i++)
            if (i < left) p[i] = from_f32<T>(x[i]);
    }
}

struct MxOut {
    uint8_t *codes, *scales;
    long long pitch, wide;          // bytes of a row, columns of a row
    int bits;
};

// Codes and scale of 8 columns from `col` on (a multiple of 8) of row r; the warp's lanes hold consecutive columns, the
// first of them a multiple of 256. All lanes call it; columns from `wide` on are not stored.
__device__ __forceinline__ void mx_store8(const MxOut &o, long long r, long long col, const float (&x)[LANE])
{
    const int lane = threadIdx.x & 31;
    // magnitudes as whole numbers keep their order, infinities and NaN above all
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < LANE; i++) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
    top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
    const bool fine = top < 0x7F800000u;
    const int e = (int)(top >> 23) - (o.bits == 4 ? 2 : 8);         // subnormals have field 0: the smallest scale
    const uint32_t s = fine ? (uint32_t)max(e, 0) : 255u;
    const float inv = __uint_as_float(fine ? (254u - s) << 23 : 0u);
    float q[LANE];
#pragma unroll
    for (int i = 0; i < LANE; i++) q[i] = fine ? x[i] * inv : 0.0f;
    uint32_t word = s << (lane >> 2 & 3) * 8;
    word |= __shfl_xor_sync(0xFFFFFFFFu, word, 4);
    word |= __shfl_xor_sync(0xFFFFFFFFu, word, 8);
    if (col >= o.wide) return;
    uint8_t *const row = o.codes + r * o.pitch;
    if (o.bits == 4) {
        uint32_t c = 0;
#pragma unroll
        for (int i = 0; i < LANE; i += 2)
            c |= (uint32_t)__nv_cvt_float2_to_fp4x2(make_float2(q[i], q[i + 1]), __NV_E2M1, cudaRoundNearest) << 4 * i;
        *(uint32_t *)(row + col / 2) = c;
    } else {
        uint32_t c[2];
#pragma unroll
        for (int i = 0; i < 2; i++)
            c[i] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(q[4 * i], q[4 * i + 1]), __NV_SATFINITE, __NV_E4M3) |
                   (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(q[4 * i + 2], q[4 * i + 3]), __NV_SATFINITE, __NV_E4M3) << 16;
        *(uint2 *)(row + col) = make_uint2(c[0], c[1]);
    }
    if ((lane & 15) == 0) *(uint32_t *)(o.scales + mx_scale_at(r, col / MX_BLOCK, o.wide / MX_ATOM)) = word;
}

// ------------------------------------------------------------------ quantisation and back

struct QuantArgs {
    const void *x;
    long long ld, cols, chunks, tasks;      // a task: 256 columns of a row
    MxOut o;
    bool vec;
};

template <typename T>
__global__ void __launch_bounds__(32 * MX_WARPS) mx_quantize_kernel(const __grid_constant__ QuantArgs p)
{
    lm_begin();
    const long long task = (long long)blockIdx.x * MX_WARPS + (threadIdx.x >> 5);
    if (task >= p.tasks) return;
    const long long r = task / p.chunks, col = (task - r * p.chunks) * 256 + (threadIdx.x & 31) * LANE;
    float x[LANE];
    load8((const T *)p.x + r * p.ld + col, p.cols - col, p.vec, x);
    mx_store8(p.o, r, col, x);
}

template <typename T>
__global__ void __launch_bounds__(32 * MX_WARPS) mx_dequantize_kernel(const __grid_constant__ QuantArgs p, T *y)
{
    lm_begin();
    const long long task = (long long)blockIdx.x * MX_WARPS + (threadIdx.x >> 5);
    if (task >= p.tasks) return;
    const long long r = task / p.chunks, col = (task - r * p.chunks) * 256 + (threadIdx.x & 31) * LANE;
    if (col >= p.cols) return;
    const uint8_t *const row = p.o.codes + r * p.o.pitch;
    const uint32_t s = p.o.scales[mx_scale_at(r, col / MX_BLOCK, p.o.wide / MX_ATOM)];
    const float scale = __uint_as_float(s == 255 ? 0x7FFFFFFFu : s ? s << 23 : 0x00400000u);
    float x[LANE];
    if (p.o.bits == 4) {
        const uint32_t c = *(const uint32_t *)(row + col / 2);
#pragma unroll
        for (int i = 0; i < LANE; i += 2) {
            const float2 v = __half22float2(__half2(__nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)(c >> 4 * i & 255), __NV_E2M1)));
            x[i] = v.x * scale, x[i + 1] = v.y * scale;
        }
    } else {
        const uint2 c = *(const uint2 *)(row + col);
#pragma unroll
        for (int i = 0; i < LANE; i += 2) {
            const uint32_t w = (i < 4 ? c.x : c.y) >> (i & 2) * 8 & 0xFFFF;
            const float2 v = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)w, __NV_E4M3)));
            x[i] = v.x * scale, x[i + 1] = v.y * scale;
        }
    }
    store8(y + r * p.ld + col, p.cols - col, p.vec, x);
}

MxOut mx_out(const tcg_mx_t &m)
{
    return { m.codes, m.scales, mx_pitch(m.cols, m.bits), mx_wide(m.cols), m.bits };
}

bool aligned16(const void *p, int64_t ld, ggml_type_t t) { return (uintptr_t)p % 16 == 0 && ld * lm_type_size(t) % 16 == 0; }

bool quant_args(const char *who, QuantArgs &p, const tcg_mx_t &m, const void *x, int64_t ld, ggml_type_t t)
{
    p.x = x;
    p.ld = ld;
    p.cols = m.cols;
    p.chunks = (mx_wide(m.cols) + 255) / 256;
    p.tasks = p.chunks * m.rows;
    p.o = mx_out(m);
    p.vec = aligned16(x, ld, t);
    if (p.tasks > 0x7fffffffll * MX_WARPS) return fail("%s: %d rows of %d columns are too many for one call", who, m.rows, m.cols);
    return true;
}

// ------------------------------------------------------------------ residual and norm

struct NormArgs {
    const void *x, *r;
    void *h, *y;
    const float *w;
    long long ldx, ldr, ldh, ldy;
    MxOut o;                        // codes NULL: none
    int rows, cols;
    double eps;
    bool vx, vr, vh, vy, vw;        // 16-byte accesses
};

// y = v * rstd * w as fp32 (round to nearest), and as the odd-rounded number that may be rounded once more.
struct Normed {
    float near, odd;
};
__device__ __forceinline__ Normed normed(float v, float r_hi, float r_lo, float w)
{
    const float q = v * r_hi, ql = fmaf(v, r_lo, fmaf(v, r_hi, -q));
    const float y = q * w, rest = fmaf(ql, w, fmaf(q, w, -y));
    // y + rest, |rest| up to an ulp: once more, so that y is the nearest
    const float near = y + rest, left = rest - (near - y);
    uint32_t b = __float_as_uint(near);
    if (left != 0.0f && (b & 0x7FFFFFFFu) < 0x7F800000u) {
        // a magnitude rounded up goes back by one, then the last bit says that something is left
        if (near != 0.0f && (__float_as_uint(left) ^ b) >> 31) b -= 1;
        b |= 1;
    }
    return { near, __uint_as_float(b) };
}

// A row's columns are dealt out to G threads (a warp's 32, or the CTA's), N pieces of 8 consecutive columns each.
template <typename T, int N, bool WARP>
__global__ void __launch_bounds__(1024) add_rms_norm_kernel(const __grid_constant__ NormArgs p)
{
    const int G = WARP ? 32 : blockDim.x, t = WARP ? threadIdx.x & 31 : threadIdx.x;
    const long long row = WARP ? (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    __shared__ double part[32];
    lm_begin();
    if (WARP && row >= p.rows) return;
    float v[N][LANE];
    double ss = 0.0;
#pragma unroll
    for (int k = 0; k < N; k++) {
        const long long col = (long long)(k * G + t) * LANE;
        load8((const T *)p.x + row * p.ldx + col, p.cols - col, p.vx, v[k]);
        if (p.r) {
            float r[LANE];
            load8((const T *)p.r + row * p.ldr + col, p.cols - col, p.vr, r);
#pragma unroll
            for (int i = 0; i < LANE; i++) v[k][i] = to_f32(from_f32<T>(v[k][i] + r[i]));
        }
    }
#pragma unroll
    for (int k = 0; k < N; k++) {
        const long long col = (long long)(k * G + t) * LANE;
        if (p.h) store8((T *)p.h + row * p.ldh + col, p.cols - col, p.vh, v[k]);
#pragma unroll
        for (int i = 0; i < LANE; i++) ss = fma((double)v[k][i], (double)v[k][i], ss);
    }
    if (!p.y && !p.o.codes) return;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
    if (!WARP) {
        if ((t & 31) == 0) part[t >> 5] = ss;
        __syncthreads();
        const int warps = blockDim.x >> 5;
        ss = (t & 31) < warps ? part[t & 31] : 0.0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
    }
    const double rstd = rsqrt(ss / p.cols + p.eps);
    const float r_hi = (float)rstd, r_lo = (float)(rstd - r_hi);
    // rows whose root leaves fp32's normal numbers take the product in 64 bits
    const bool plain = rstd > 1e-30 && rstd < 1e30;
#pragma unroll
    for (int k = 0; k < N; k++) {
        const long long col = (long long)(k * G + t) * LANE;
        float w[LANE], near[LANE], odd[LANE];
        load8(p.w + col, p.cols - col, p.vw, w);
#pragma unroll
        for (int i = 0; i < LANE; i++) {
            if (plain) {
                const Normed n = normed(v[k][i], r_hi, r_lo, w[i]);
                near[i] = n.near, odd[i] = n.odd;
            } else {
                const double y = v[k][i] * rstd * w[i];
                near[i] = (float)y;
                odd[i] = __double2float_rz(y);
                if ((double)odd[i] != y && fabsf(near[i]) < INFINITY) odd[i] = __uint_as_float(__float_as_uint(odd[i]) | 1);
                else odd[i] = fabsf(near[i]) < INFINITY ? odd[i] : near[i];
            }
            if (col + i >= p.cols) near[i] = odd[i] = 0.0f;         // 0 * rstd may be NaN there
        }
        if (p.y) store8((T *)p.y + row * p.ldy + col, p.cols - col, p.vy, sizeof(T) == 4 ? near : odd);
        if (p.o.codes) mx_store8(p.o, row, col, odd);
    }
}

template <typename T, int N, bool WARP>
bool norm_launch(const NormArgs &p, int threads)
{
    const unsigned grid = WARP ? ceil_div(p.rows, threads / 32) : (unsigned)p.rows;
    TCG_CUDA(launch_pdl(add_rms_norm_kernel<T, N, WARP>, dim3(grid), dim3(threads), 0, ctx().cur, p));
    return true;
}

template <typename T>
bool norm_go(const NormArgs &p)
{
    const int pieces = (int)(mx_wide(p.cols) / LANE);           // of 8 columns, those behind the last one included
    if (pieces <= 32) return norm_launch<T, 1, true>(p, 256);
    if (pieces <= 64) return norm_launch<T, 2, true>(p, 256);
    const int n = pieces <= 1024 ? 1 : pieces <= 2048 ? 2 : 4;
    const int threads = ((pieces + n - 1) / n + 31) / 32 * 32;
    if (n == 1) return norm_launch<T, 1, false>(p, threads);
    if (n == 2) return norm_launch<T, 2, false>(p, threads);
    return norm_launch<T, 4, false>(p, threads);
}

}  // namespace
}  // namespace tcg

using namespace tcg;

extern "C" size_t tcg_mx_code_bytes(int rows, int cols, int bits)
{
    if (rows < 0 || rows > TCG_MX_MAX_ROWS || cols < 1 || cols > TCG_MX_MAX_COLS || (bits != 4 && bits != 8)) return 0;
    return (size_t)rows * (size_t)mx_pitch(cols, bits);
}

extern "C" size_t tcg_mx_scale_bytes(int rows, int cols)
{
    if (rows < 0 || rows > TCG_MX_MAX_ROWS || cols < 1 || cols > TCG_MX_MAX_COLS) return 0;
    return (size_t)(rows + MX_ATOM - 1) / MX_ATOM * MX_ATOM * (size_t)(mx_wide(cols) / MX_BLOCK);
}

extern "C" bool tcg_mx_quantize(const tcg_mx_t *m, const void *x, int64_t ld, ggml_type_t t)
{
    const char *who = "tcg_mx_quantize";
    if (!lm_type_size(t)) return fail("%s: type %d is not F32, F16 or BF16", who, (int)t);
    if (!mx_check(who, "matrix", m) || !mx_rows(who, "x", x, m->rows, m->cols, ld, t)) return false;
    if (!lm_ready(who)) return false;
    if (!m->rows) return true;
    QuantArgs p = {};
    if (!quant_args(who, p, *m, x, ld, t)) return false;
    return lm_by_type(t, [&](auto v) {
        TCG_CUDA(launch_pdl(mx_quantize_kernel<decltype(v)>, dim3(ceil_div(p.tasks, MX_WARPS)), dim3(32 * MX_WARPS), 0, ctx().cur, p));
        return true;
    });
}

extern "C" bool tcg_mx_dequantize(void *y, const tcg_mx_t *m, int64_t ld, ggml_type_t t)
{
    const char *who = "tcg_mx_dequantize";
    if (!lm_type_size(t)) return fail("%s: type %d is not F32, F16 or BF16", who, (int)t);
    if (!mx_check(who, "matrix", m) || !mx_rows(who, "y", y, m->rows, m->cols, ld, t)) return false;
    if (!lm_ready(who)) return false;
    if (!m->rows) return true;
    QuantArgs p = {};
    if (!quant_args(who, p, *m, y, ld, t)) return false;
    return lm_by_type(t, [&](auto v) {
        using T = decltype(v);
        TCG_CUDA(launch_pdl(mx_dequantize_kernel<T>, dim3(ceil_div(p.tasks, MX_WARPS)), dim3(32 * MX_WARPS), 0, ctx().cur, p, (T *)y));
        return true;
    });
}

extern "C" bool tcg_add_rms_norm(void *h, void *y, const tcg_mx_t *mx, const void *x, const void *r, const float *w, float eps,
                                 int n_tok, int cols, int64_t ld_h, int64_t ld_y, int64_t ld_x, int64_t ld_r, ggml_type_t t)
{
    const char *who = "tcg_add_rms_norm";
    if (!lm_type_size(t)) return fail("%s: type %d is not F32, F16 or BF16", who, (int)t);
    if (n_tok < 0 || cols < 1 || cols > TCG_NORM_MAX_COLS)
        return fail("%s: %d rows of %d columns (at most %d)", who, n_tok, cols, TCG_NORM_MAX_COLS);
    if (!(eps >= 0.0f) || eps > 1e30f) return fail("%s: eps %g", who, (double)eps);
    if (mx && (!mx_check(who, "mx", mx) || mx->rows != n_tok || mx->cols != cols)) {
        if (mx->rows != n_tok || mx->cols != cols)
            return fail("%s: mx of %d rows and %d columns for %d rows of %d", who, mx->rows, mx->cols, n_tok, cols);
        return false;
    }
    if (!h && !y && !mx) return fail("%s: no output", who);
    if (n_tok) {
        if (!mx_rows(who, "x", x, n_tok, cols, ld_x, t) || (r && !mx_rows(who, "r", r, n_tok, cols, ld_r, t)) ||
            (h && !mx_rows(who, "h", h, n_tok, cols, ld_h, t)) || (y && !mx_rows(who, "y", y, n_tok, cols, ld_y, t)))
            return false;
        if ((y || mx) && (!w || (uintptr_t)w % 4)) return fail("%s: no weights, or misaligned ones", who);
    }
    if (!lm_ready(who)) return false;
    if (!n_tok) return true;
    NormArgs p = {};
    p.x = x, p.r = r, p.h = h, p.y = y, p.w = w;
    p.ldx = ld_x, p.ldr = ld_r, p.ldh = ld_h, p.ldy = ld_y;
    if (mx) p.o = mx_out(*mx);
    p.rows = n_tok, p.cols = cols;
    p.eps = eps;
    p.vx = aligned16(x, ld_x, t), p.vr = aligned16(r, ld_r, t), p.vh = aligned16(h, ld_h, t), p.vy = aligned16(y, ld_y, t);
    p.vw = (uintptr_t)w % 16 == 0;
    return lm_by_type(t, [&](auto v) { return norm_go<decltype(v)>(p); });
}
