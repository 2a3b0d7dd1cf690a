// mx.cu -- microscaled matrices: tcg_mx_quantize, tcg_mx_dequantize, and the residual's addition with the
// root-mean-square norm whose rows come out in 8 or 4 bits (tcg_add_rms_norm).
//
// A block of 32 columns has the scale 2^s, s = floor(log2 max|x|) - m, m = 2 for E2M1 (largest value 6 = 1.5 * 2^2) and 8
// for E4M3 (448 = 1.75 * 2^8), and codes rn(x / 2^s). floor(log2) is the exponent field of the largest magnitude, and the
// division by a power of two is exact, so codes are the format's nearest values to the inputs themselves.
//
// The norm's codes have to be those of y = h / sqrt(mean(h^2) + eps) * w, not of an fp32 approximation that may lie on
// the other side of the border between two codes. The sum of squares and the root are taken in 64 bits; the products in
// fp32, within 2^-21 of y. Where y (1 - 2^-21) and y (1 + 2^-21) have the same code, that is y's (rounding keeps order);
// where they have not (one value in 2^16 or so), the warp takes its values again in 64 bits, cut to fp32 with the last bit odd
// where a rest is left: rounding that once more cannot meet a tie that is none.
//
// All three are bound by memory: 14336 x 4096 fp32 values quantised to 4 bits in 39 us (6.8 TB/s), read back to bf16 in
// 25.2 us (5.9 TB/s, what a fill of the same bytes reaches); 4096 rows of 4096 fp32 values with their residual to 8 bits in
// 38.6 us (5.7 TB/s: its second pass over the row waits for the sum). One token's norm takes 2.7 us, 1.8 of them the launch.
#include "mx.cuh"

#include <cuda_fp4.h>
#include <cuda_fp8.h>

#include <string.h>

#include <type_traits>

namespace tcg {
namespace {

constexpr int LANE = 8;             // consecutive columns of a lane: 4 lanes make a block, 16 a word of scales
constexpr int MX_WARPS = 4;         // of a CTA (1501 rows of 4100 16-bit values, 4103 apart, to 4 bits 5.7 us, with 8 5.9)

// 8 elements as they are held.
template <typename T>
struct Raw {
    static constexpr int W = 2 * sizeof(T);     // words
    uint32_t w[W];
    __device__ __forceinline__ T at(int i) const
    {
        T v;
        if constexpr (sizeof(T) == 4) memcpy(&v, &w[i], 4);
        else {
            const unsigned short h = (unsigned short)(w[i / 2] >> (i & 1) * 16);
            memcpy(&v, &h, 2);
        }
        return v;
    }
    __device__ __forceinline__ void set(int i, T v)
    {
        if constexpr (sizeof(T) == 4) memcpy(&w[i], &v, 4);
        else {
            unsigned short h;
            memcpy(&h, &v, 2);
            w[i / 2] = i & 1 ? (w[i / 2] & 0xFFFFu) | (uint32_t)h << 16 : h;
        }
    }
};

// Words k[0 .. N - 1] of the bytes that start at byte `off` (0 .. 15) of k[0 .. N + 3].
template <int N>
__device__ __forceinline__ void shift_bytes(uint32_t (&k)[N + 4], uint32_t off)
{
#pragma unroll
    for (int i = 0; i < N + 2; i++) k[i] = off & 8 ? k[i + 2] : k[i];
#pragma unroll
    for (int i = 0; i < N + 1; i++) k[i] = off & 4 ? k[i + 1] : k[i];
#pragma unroll
    for (int i = 0; i < N; i++) k[i] = __funnelshift_r(k[i], k[i + 1], (off & 3) * 8);
}

// A lane's 8 elements of a row, of which `left` exist (the others are 0). A row that starts on no 8-byte boundary is read
// by the aligned 16-byte words around it and shifted, where those lie in [lo, hi), the array (1501 rows of 4100 quantised: 6.4 us, element by element 8.1).
// VEC: rows start on 16-byte boundaries.
template <bool VEC, typename T>
__device__ __forceinline__ Raw<T> load_row(const T *p, long long left, const void *lo, const void *hi)
{
    constexpr int W = Raw<T>::W;
    Raw<T> r;
    const uintptr_t at = (uintptr_t)p;
    const uint32_t off = VEC ? 0 : (uint32_t)at & 15;
    if (left >= LANE) {
        if (VEC || off == 0) {
#pragma unroll
            for (int i = 0; i < W; i += 4) {
                const uint4 v = ((const uint4 *)p)[i / 4];
                r.w[i] = v.x, r.w[i + 1] = v.y, r.w[i + 2] = v.z, r.w[i + 3] = v.w;
            }
            return r;
        }
        if (off == 8) {
#pragma unroll
            for (int i = 0; i < W; i += 2) {
                const uint2 v = ((const uint2 *)p)[i / 2];
                r.w[i] = v.x, r.w[i + 1] = v.y;
            }
            return r;
        }
        const uint4 *const from = (const uint4 *)(at - off);
        if (!VEC && (const void *)from >= lo && (const void *)(from + W / 4 + 1) <= hi) {
            uint32_t k[W + 4];
#pragma unroll
            for (int i = 0; i < W + 4; i += 4) {
                const uint4 v = from[i / 4];
                k[i] = v.x, k[i + 1] = v.y, k[i + 2] = v.z, k[i + 3] = v.w;
            }
            shift_bytes<W>(k, off);
#pragma unroll
            for (int i = 0; i < W; i++) r.w[i] = k[i];
            return r;
        }
    }
#pragma unroll
    for (int i = 0; i < LANE; i++) r.set(i, i < left ? p[i] : from_f32<T>(0.0f));
    return r;
}

// The same back; all lanes of a warp call it, on consecutive elements of one row. Off an 8-byte boundary a lane writes the
// aligned words that start in the lane before it, with that lane's last bytes.
template <bool VEC, typename T>
__device__ __forceinline__ void store_row(T *p, long long left, const Raw<T> &r)
{
    constexpr int W = Raw<T>::W;
    const uintptr_t at = (uintptr_t)p;
    const uint32_t off = VEC ? 0 : (uint32_t)at & 15;
    const bool full = left >= LANE;
    if (VEC || off == 0 || off == 8) {
        if (full && (VEC || off == 0)) {
#pragma unroll
            for (int i = 0; i < W; i += 4) ((uint4 *)p)[i / 4] = make_uint4(r.w[i], r.w[i + 1], r.w[i + 2], r.w[i + 3]);
        } else if (full) {
#pragma unroll
            for (int i = 0; i < W; i += 2) ((uint2 *)p)[i / 2] = make_uint2(r.w[i], r.w[i + 1]);
        } else if (left > 0) {
#pragma unroll
            for (int i = 0; i < LANE; i++)
                if (i < left) p[i] = r.at(i);
        }
        return;
    }
    const int lane = threadIdx.x & 31;
    const unsigned fulls = __ballot_sync(0xFFFFFFFFu, full);
    uint32_t k[W + 4];
#pragma unroll
    for (int i = 0; i < 4; i++) k[i] = __shfl_up_sync(0xFFFFFFFFu, r.w[W - 4 + i], 1);
    const bool before = lane > 0 && (fulls >> (lane - 1) & 1), after = lane < 31 && (fulls >> (lane + 1) & 1);
#pragma unroll
    for (int i = 0; i < W; i++) k[4 + i] = r.w[i];
    shift_bytes<W>(k, 16 - off);
    uint4 *const words = (uint4 *)(at - off);
    if (full) {
        if (before) words[0] = make_uint4(k[0], k[1], k[2], k[3]);
#pragma unroll
        for (int i = 4; i < W; i += 4) words[i / 4] = make_uint4(k[i], k[i + 1], k[i + 2], k[i + 3]);
        if (before && after) return;
    }
    // what no word of this lane or the next one holds
    const int to = !full ? (int)max(left, 0ll) : before ? 0 : (int)((16 - off) / sizeof(T));
    const int from = full && !after ? LANE - (int)(off / sizeof(T)) : LANE;
#pragma unroll
    for (int i = 0; i < LANE; i++)
        if (i < to || i >= from) p[i] = r.at(i);
}

// A word's two 16-bit values, and back; a word is one fp32 value.
__device__ __forceinline__ float2 pair_f32(uint32_t w, __half)
{
    __half2 h;
    memcpy(&h, &w, 4);
    return __half22float2(h);
}
__device__ __forceinline__ float2 pair_f32(uint32_t w, __nv_bfloat16) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }
__device__ __forceinline__ uint32_t pair_word(float a, float b, __half)
{
    const __half2 h = __floats2half2_rn(a, b);
    uint32_t w;
    memcpy(&w, &h, 4);
    return w;
}
__device__ __forceinline__ uint32_t pair_word(float a, float b, __nv_bfloat16)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    uint32_t w;
    memcpy(&w, &h, 4);
    return w;
}

template <typename T>
__device__ __forceinline__ void unpack(const Raw<T> &r, float (&x)[LANE])
{
#pragma unroll
    for (int i = 0; i < Raw<T>::W; i++) {
        if constexpr (sizeof(T) == 4) x[i] = __uint_as_float(r.w[i]);
        else {
            const float2 v = pair_f32(r.w[i], T());
            x[2 * i] = v.x, x[2 * i + 1] = v.y;
        }
    }
}
template <typename T>
__device__ __forceinline__ Raw<T> packed(const float (&x)[LANE])
{
    Raw<T> r;
#pragma unroll
    for (int i = 0; i < Raw<T>::W; i++) {
        if constexpr (sizeof(T) == 4) r.w[i] = __float_as_uint(x[i]);
        else r.w[i] = pair_word(x[2 * i], x[2 * i + 1], T());
    }
    return r;
}

struct MxOut {
    uint8_t *codes, *scales;
    long long pitch, wide;          // bytes of a row, columns of a row
    int bits;
};

// The scale byte of a block, from the bits of its largest magnitude (infinities and NaN above all), and 1 / scale (0 for a
// block that is NaN). Subnormals have exponent field 0: the smallest scale.
__device__ __forceinline__ uint32_t mx_scale(uint32_t top, int bits)
{
    return top < 0x7F800000u ? (uint32_t)max((int)(top >> 23) - (bits == 4 ? 2 : 8), 0) : 255u;
}
__device__ __forceinline__ float mx_inverse(uint32_t s) { return __uint_as_float(s == 255 ? 0u : (254u - s) << 23); }
// maxima that a NaN wins
__device__ __forceinline__ float max_nan(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ uint32_t mx_top(const float (&x)[LANE])
{
    float t = max_nan(fabsf(x[0]), fabsf(x[1]), fabsf(x[2]));
    t = max_nan(t, fabsf(x[3]), fabsf(x[4]));
    t = max_nan(t, fabsf(x[5]), fabsf(x[6]));
    t = max_nan(t, fabsf(x[7]));
    t = max_nan(t, __shfl_xor_sync(0xFFFFFFFFu, t, 1));
    return __float_as_uint(max_nan(t, __shfl_xor_sync(0xFFFFFFFFu, t, 2))) & 0x7FFFFFFFu;
}
__device__ __forceinline__ uint2 mx_codes(const float (&q)[LANE], int bits)
{
    uint2 c = make_uint2(0, 0);
    if (bits == 4) {
        asm("{\n\t.reg .b8 a, b, c, d;\n\t"
            "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
            "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
            "mov.b32 %0, {a, b, c, d};\n\t}"
            : "=r"(c.x) : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]), "f"(q[4]), "f"(q[5]), "f"(q[6]), "f"(q[7]));
    } else {
        asm("{\n\t.reg .b16 a, b, c, d;\n\t"
            "cvt.rn.satfinite.e4m3x2.f32 a, %3, %2;\n\tcvt.rn.satfinite.e4m3x2.f32 b, %5, %4;\n\t"
            "cvt.rn.satfinite.e4m3x2.f32 c, %7, %6;\n\tcvt.rn.satfinite.e4m3x2.f32 d, %9, %8;\n\t"
            "mov.b32 %0, {a, b};\n\tmov.b32 %1, {c, d};\n\t}"
            : "=r"(c.x), "=r"(c.y)
            : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]), "f"(q[4]), "f"(q[5]), "f"(q[6]), "f"(q[7]));
    }
    return c;
}
// A lane's codes to row r, column `col` (not from `wide` on); returns the four scales of the 128 columns it is among.
__device__ __forceinline__ uint32_t mx_put(const MxOut &o, long long r, long long col, uint2 c, uint32_t s)
{
    uint32_t word = s << (threadIdx.x >> 2 & 3) * 8;
    word |= __shfl_xor_sync(0xFFFFFFFFu, word, 4);
    word |= __shfl_xor_sync(0xFFFFFFFFu, word, 8);
    if (col < o.wide) {
        uint8_t *const row = o.codes + r * o.pitch;
        if (o.bits == 4) *(uint32_t *)(row + col / 2) = c.x;
        else *(uint2 *)(row + col) = c;
    }
    return word;
}

// 8 columns from `col` on (a multiple of 8) of row r; the warp's lanes hold consecutive columns, the first of them a multiple
// of 256. All lanes call it.
__device__ __forceinline__ uint32_t mx_store8(const MxOut &o, long long r, long long col, const float (&x)[LANE])
{
    const uint32_t s = mx_scale(mx_top(x), o.bits);
    const float inv = mx_inverse(s);
    float q[LANE];
#pragma unroll
    for (int i = 0; i < LANE; i++) q[i] = x[i] * inv;
    return mx_put(o, r, col, mx_codes(q, o.bits), s);
}

// The same for values known to within 2^-22 of themselves (an infinity may be a number that was rounded up): false (and
// nothing stored) where some lane's codes or scales depend on more than that.
__device__ __forceinline__ bool mx_store8_near(const MxOut &o, long long r, long long col, const float (&x)[LANE], uint32_t &word)
{
    constexpr float LOW = 1.0f - 0x1p-21f, HIGH = 1.0f + 0x1p-21f;
    const uint32_t top = mx_top(x);
    const uint32_t s = mx_scale(__float_as_uint(__uint_as_float(min(top, 0x7F7FFFFFu)) * LOW), o.bits);
    const float low = mx_inverse(s) * LOW, high = mx_inverse(s) * HIGH;     // inverse is a power of two: both are exact
    float q[LANE];
#pragma unroll
    for (int i = 0; i < LANE; i++) q[i] = x[i] * low;
    const uint2 c = mx_codes(q, o.bits);
#pragma unroll
    for (int i = 0; i < LANE; i++) q[i] = x[i] * high;
    const uint2 d = mx_codes(q, o.bits);
    const bool sure = ((c.x ^ d.x) | (c.y ^ d.y)) == 0 && s == mx_scale(__float_as_uint(__uint_as_float(top) * HIGH), o.bits);
    if (!__all_sync(0xFFFFFFFFu, sure)) return false;
    word = mx_put(o, r, col, c, s);
    return true;
}

// ------------------------------------------------------------------ quantisation and back

// A warp takes 256 columns of the rows l, l + 32, l + 64 and l + 96 of a group of 128: their scales are 16 bytes in one
// place, and four rows' loads are under way together.
struct QuantArgs {
    void *x;
    const void *end;                // of x
    long long ld, cols;
    unsigned rows, chunks, tasks;
    MxOut o;
    bool vec;
};

struct QuantTask {
    unsigned group, line;
    long long col;
    bool live;
};
__device__ __forceinline__ QuantTask quant_task(const QuantArgs &p)
{
    const unsigned task = blockIdx.x * MX_WARPS + (threadIdx.x >> 5), row = task / p.chunks;
    return { row / 32, row % 32, (long long)(task - row * p.chunks) * 256 + (threadIdx.x & 31) * LANE, task < p.tasks };
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(32 * MX_WARPS) mx_quantize_kernel(const __grid_constant__ QuantArgs p)
{
    lm_begin();
    const QuantTask t = quant_task(p);
    const unsigned first = t.group * 128 + t.line;
    if (!t.live || first >= p.rows) return;
    Raw<T> raw[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const long long r = first + 32 * i;
        raw[i] = load_row<VEC>((const T *)p.x + r * p.ld + t.col, r < p.rows ? p.cols - t.col : 0, p.x, p.end);
    }
    uint32_t word[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const long long r = first + 32 * i;
        if (r >= p.rows) break;
        float x[LANE];
        unpack(raw[i], x);
        word[i] = mx_store8(p.o, r, t.col, x);
    }
    if ((threadIdx.x & 15) || t.col >= p.o.wide) return;
    uint32_t *const at = (uint32_t *)(p.o.scales + mx_scale_at(first, t.col / MX_BLOCK, p.o.wide / MX_ATOM));
    if (first + 96 < p.rows) *(uint4 *)at = make_uint4(word[0], word[1], word[2], word[3]);
    else
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (first + 32 * i < p.rows) at[i] = word[i];
}

// C times 256 columns a warp, so that more than one row's 128 bytes of codes and its scales are under way. Ten CTAs' registers
// of an SM for aligned rows, with two chunks at the price of 24 bytes spilled: 14336 x 4096 from 4 bits to bf16 25.1 us, nine
// 25.7, twelve (with more spills) 30.2.
template <typename T, int C, bool VEC>
__global__ void __launch_bounds__(32 * MX_WARPS, VEC ? 10 : 1) mx_dequantize_kernel(const __grid_constant__ QuantArgs p)
{
    lm_begin();
    QuantTask t = quant_task(p);
    t.col = (t.col - (threadIdx.x & 31) * LANE) * C + (threadIdx.x & 31) * LANE;
    const unsigned first = t.group * 128 + t.line;
    if (!t.live || first >= p.rows) return;
    uint2 code[C][4];
    uint4 scales[C];
#pragma unroll
    for (int c = 0; c < C; c++) {
        const long long col = t.col + 256 * c;
        const bool in = col < p.o.wide;
        scales[c] = make_uint4(0, 0, 0, 0);
        if (in) scales[c] = *(const uint4 *)(p.o.scales + mx_scale_at(first, col / 128 * 4, p.o.wide / MX_ATOM));
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const long long r = first + 32 * i;
            code[c][i] = make_uint2(0, 0);
            if (in && r < p.rows) {
                if (p.o.bits == 4) code[c][i].x = *(const uint32_t *)(p.o.codes + r * p.o.pitch + col / 2);
                else code[c][i] = *(const uint2 *)(p.o.codes + r * p.o.pitch + col);
            }
        }
    }
#pragma unroll
    for (int c = 0; c < C; c++) {
        const long long col = t.col + 256 * c;
        const uint32_t words[4] = { scales[c].x, scales[c].y, scales[c].z, scales[c].w };
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const long long r = first + 32 * i;
            if (r >= p.rows) break;
            const uint32_t s = words[i] >> (threadIdx.x >> 2 & 3) * 8 & 255;
            const float scale = __uint_as_float(s == 255 ? 0x7FFFFFFFu : s ? s << 23 : 0x00400000u);
            float x[LANE];
            if (p.o.bits == 4) {
#pragma unroll
                for (int j = 0; j < LANE; j += 2) {
                    const __half2_raw h = __nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)(code[c][i].x >> 4 * j & 255), __NV_E2M1);
                    const float2 v = __half22float2(__half2(h));
                    x[j] = v.x * scale, x[j + 1] = v.y * scale;
                }
            } else {
#pragma unroll
                for (int j = 0; j < LANE; j += 2) {
                    const uint32_t w = (j < 4 ? code[c][i].x : code[c][i].y) >> (j & 2) * 8 & 0xFFFF;
                    const float2 v = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)w, __NV_E4M3)));
                    x[j] = v.x * scale, x[j + 1] = v.y * scale;
                }
            }
            store_row<VEC>((T *)p.x + r * p.ld + col, p.cols - col, packed<T>(x));
        }
    }
}

MxOut mx_out(const tcg_mx_t &m)
{
    return { m.codes, m.scales, mx_pitch(m.cols, m.bits), mx_wide(m.cols), m.bits };
}

// Whether every row starts on a 16-byte boundary.
bool on_16(const void *p, int64_t ld, ggml_type_t t) { return (uintptr_t)p % 16 == 0 && ld * (int64_t)lm_type_size(t) % 16 == 0; }

bool quant_args(const char *who, QuantArgs &p, const tcg_mx_t &m, void *x, int64_t ld, ggml_type_t t, int wide = 1)
{
    p.x = x;
    p.end = (const char *)x + ((m.rows - 1) * ld + m.cols) * (int64_t)lm_type_size(t);
    p.ld = ld;
    p.cols = m.cols;
    p.rows = (unsigned)m.rows;
    p.chunks = (unsigned)((mx_wide(m.cols) + 256 * wide - 1) / (256 * wide));
    // rows beyond 128 are dealt out by groups, 32 lines each; a few rows are lines of one group
    const long long lines = m.rows < 32 ? m.rows : (m.rows + 127ll) / 128 * 32, tasks = lines * p.chunks;
    if (tasks > 0x7fffffffll) return fail("%s: %d rows of %d columns are too many for one call", who, m.rows, m.cols);
    p.tasks = (unsigned)tasks;
    p.o = mx_out(m);
    p.vec = on_16(x, ld, t);
    return true;
}

// ------------------------------------------------------------------ residual and norm

struct NormArgs {
    const void *x, *r;
    const void *x_end, *r_end;      // of the arrays
    void *h, *y;
    const float *w;
    long long ldx, ldr, ldh, ldy;
    MxOut o;                        // codes NULL: none
    int rows, cols;
    double eps, mean;               // 1 / cols
    bool vec_in, vec_out;
};

// v * rstd * w from 64 bits, cut to fp32 with its last bit odd where something is left. (Infinities and NaN as they are.)
__device__ __forceinline__ float normed_odd(float v, double rstd, float w)
{
    const double d = v * rstd * w;
    if (!(fabs(d) <= 0x1.fffffep+127)) return (float)d;
    const float y = __double2float_rz(d);
    return (double)y == d ? y : __uint_as_float(__float_as_uint(y) | 1);
}

// A row's columns are dealt out to G threads (a warp's 32, or the CTA's, at most MOST), N pieces of 8 consecutive columns each.
// CTAs an SM that registers are kept for. 4096 rows of 4096 fp32 values with their residual, to 8 bits: two pieces a thread of 256
// and four CTAs 38.6 us (5.7 TB/s), five (with spills) 40.3; two of 512 and two CTAs 40.9; one of 512 and three 43.2; four of 128
// and five 50.0. Without codes five fit. 512 bf16 rows of 16384 without codes: two CTAs 16.5 us, one (76 registers) 19.9. Four
// pieces of 1024 (more than 16384 columns) have 64 registers by the block's size, and fp32 rows spill 80 bytes, up to 376 with
// codes off 16-byte boundaries: 256 rows of 32768 with their residual 31.9 us (4.2 TB/s), in bf16 18.2.
constexpr int norm_ctas(int size, int n, int most, bool mx)
{
    return n == 2 && most == 256 ? mx ? 4 : 5 : n == 4 && most == 512 && size == 2 && !mx ? 2 : 1;
}

// VIN, VOUT: rows of x, r and w, and of h and y, start on 16-byte boundaries. MX: there are codes to write.
template <typename T, int N, int MOST, bool VIN, bool VOUT, bool MX>
__global__ void __launch_bounds__(MOST == 32 ? 256 : MOST, norm_ctas(sizeof(T), N, MOST, MX)) add_rms_norm_kernel(const __grid_constant__ NormArgs p)
{
    constexpr bool WARP = MOST == 32;
    const int G = WARP ? 32 : blockDim.x, t = WARP ? threadIdx.x & 31 : threadIdx.x;
    const long long row = WARP ? (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    __shared__ double part[32];
    lm_begin();
    if (WARP && row >= p.rows) return;
    Raw<T> h[N], r[N];
#pragma unroll
    for (int k = 0; k < N; k++) {
        const long long col = (long long)(k * G + t) * LANE;
        h[k] = load_row<VIN>((const T *)p.x + row * p.ldx + col, p.cols - col, p.x, p.x_end);
        if (p.r) r[k] = load_row<VIN>((const T *)p.r + row * p.ldr + col, p.cols - col, p.r, p.r_end);
    }
    // a thread of one piece has the registers to ask for its weights now
    Raw<float> w0;
    if (N == 1 && p.w) w0 = load_row<VIN>(p.w + (long long)t * LANE, p.cols - (long long)t * LANE, p.w, p.w + p.cols);
    double ss = 0.0;
    uint32_t low = 0xFFFFFFFFu;         // the smallest magnitude but for zeros, as twice its bits less one
#pragma unroll
    for (int k = 0; k < N; k++) {
        float v[LANE];
        unpack(h[k], v);
        if (p.r) {
            float u[LANE];
            unpack(r[k], u);
#pragma unroll
            for (int i = 0; i < LANE; i++) v[i] += u[i];
            h[k] = packed<T>(v);
            unpack(h[k], v);
        }
#pragma unroll
        for (int i = 0; i < LANE; i++) ss = fma((double)v[i], (double)v[i], ss);
        if (!std::is_same<T, __half>::value)
#pragma unroll
            for (int i = 0; i < LANE; i++) low = min(low, 2 * __float_as_uint(v[i]) - 1);
    }
    if (p.h)
#pragma unroll
        for (int k = 0; k < N; k++) {
            const long long col = (long long)(k * G + t) * LANE;
            store_row<VOUT>((T *)p.h + row * p.ldh + col, p.cols - col, h[k]);
        }
    if (!MX && !p.y) return;
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
    const double rstd = rsqrt(fma(ss, p.mean, p.eps));
    const float r_hi = (float)rstd;
    // Rows whose root leaves fp32's normal numbers take the products in 64 bits. So does a warp that holds a value, but for
    // zeros, which is so small beside its row that v * r_hi, below 2^-100, may lose bits before a large weight brings it back.
    // (f16's smallest value is 2^-40 of its largest. Lanes that choose for themselves: 4096 x 4096 bf16 24.8 us, warps 24.2.)
    const bool plain = rstd > 1e-30 && rstd < 1e30, tiny = __uint_as_float(low >> 1) * r_hi < 0x1p-100f;
    const bool fast = plain && (std::is_same<T, __half>::value || !__any_sync(0xFFFFFFFFu, tiny));
#pragma unroll
    for (int k = 0; k < N; k++) {
        const long long col = (long long)(k * G + t) * LANE;
        const Raw<float> w = N == 1 ? w0 : load_row<VIN>(p.w + col, p.cols - col, p.w, p.w + p.cols);
        float v[LANE], y[LANE];
        unpack(h[k], v);
        if (fast) {
#pragma unroll
            for (int i = 0; i < LANE; i++) y[i] = v[i] * r_hi * w.at(i);
        } else {
#pragma unroll
            for (int i = 0; i < LANE; i++) y[i] = (float)(v[i] * rstd * w.at(i));
        }
        if (col + LANE > p.cols)
#pragma unroll
            for (int i = 0; i < LANE; i++)
                if (col + i >= p.cols) y[i] = 0.0f;                 // 0 * rstd may be NaN there
        if (p.y) store_row<VOUT>((T *)p.y + row * p.ldy + col, p.cols - col, packed<T>(y));
        if (!MX) continue;
        uint32_t word;
        if (!plain || !mx_store8_near(p.o, row, col, y, word)) {
#pragma unroll
            for (int i = 0; i < LANE; i++) {
                y[i] = normed_odd(v[i], rstd, w.at(i));
                if (col + i >= p.cols) y[i] = 0.0f;
            }
            word = mx_store8(p.o, row, col, y);
        }
        if ((t & 15) == 0 && col < p.o.wide)
            *(uint32_t *)(p.o.scales + mx_scale_at(row, col / MX_BLOCK, p.o.wide / MX_ATOM)) = word;
    }
}

template <typename T, int N, int MOST>
bool norm_launch(const NormArgs &p, int threads)
{
    const unsigned grid = MOST == 32 ? ceil_div(p.rows, threads / 32) : (unsigned)p.rows;
    const auto launch = [&](auto vin, auto vout, auto codes) {
        constexpr auto fn = add_rms_norm_kernel<T, N, MOST, decltype(vin)::value, decltype(vout)::value, decltype(codes)::value>;
        return launch_pdl(fn, dim3(grid), dim3(threads), 0, ctx().cur, p);
    };
    const auto by_codes = [&](auto vin, auto vout) {
        return p.o.codes ? launch(vin, vout, std::true_type()) : launch(vin, vout, std::false_type());
    };
    const std::true_type yes;
    const std::false_type no;
    TCG_CUDA(!p.vec_in ? by_codes(no, no) : p.vec_out ? by_codes(yes, yes) : by_codes(yes, no));
    return true;
}

template <typename T>
bool norm_go(const NormArgs &p)
{
    const int pieces = (int)(mx_wide(p.cols) / LANE);           // of 8 columns, those behind the last one included
    // Few rows: a thread has one piece. Many: more, whose loads are under way together, and a join of fewer warps.
    const bool many = p.rows >= 2 * ctx().sms;
    auto threads = [&](int n) { return ((pieces + n - 1) / n + 31) / 32 * 32; };
    if (pieces <= 32) return norm_launch<T, 1, 32>(p, 256);
    if (many) {
        if (pieces <= 64) return norm_launch<T, 2, 32>(p, 256);
        if (pieces <= 512) return norm_launch<T, 2, 256>(p, threads(2));
        if (pieces <= 1024) return norm_launch<T, 2, 512>(p, threads(2));
    }
    if (pieces <= 1024) return norm_launch<T, 1, 1024>(p, threads(1));
    if (pieces <= 2048) return norm_launch<T, 4, 512>(p, threads(4));
    return norm_launch<T, 4, 1024>(p, threads(4));
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
    if (!quant_args(who, p, *m, (void *)x, ld, t)) return false;
    return lm_by_type(t, [&](auto v) {
        void (*fn)(const QuantArgs) = p.vec ? mx_quantize_kernel<decltype(v), true> : mx_quantize_kernel<decltype(v), false>;
        TCG_CUDA(launch_pdl(fn, dim3(ceil_div(p.tasks, MX_WARPS)), dim3(32 * MX_WARPS), 0, ctx().cur, p));
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
    // two chunks of columns a warp where that leaves 16 warps an SM
    const bool wide = (long long)m->rows * m->cols >= (long long)ctx().sms * 16 * 2048;
    if (!quant_args(who, p, *m, y, ld, t, wide ? 2 : 1)) return false;
    return lm_by_type(t, [&](auto v) {
        using T = decltype(v);
        void (*fn)(const QuantArgs) = p.vec ? (wide ? mx_dequantize_kernel<T, 2, true> : mx_dequantize_kernel<T, 1, true>)
                                            : (wide ? mx_dequantize_kernel<T, 2, false> : mx_dequantize_kernel<T, 1, false>);
        TCG_CUDA(launch_pdl(fn, dim3(ceil_div(p.tasks, MX_WARPS)), dim3(32 * MX_WARPS), 0, ctx().cur, p));
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
        // In place, a row's results must fall on the row itself.
        const auto in_place = [&](const void *o, int64_t ld) {
            return !o || n_tok == 1 || ((o != x || ld == ld_x) && (o != r || ld == ld_r));
        };
        if (h && h == y) return fail("%s: h and y are the same rows", who);
        if (!in_place(h, ld_h) || !in_place(y, ld_y)) return fail("%s: in place with another stride", who);
        if ((y || mx) && (!w || (uintptr_t)w % 4)) return fail("%s: no weights, or misaligned ones", who);
    }
    if (!lm_ready(who)) return false;
    if (!n_tok) return true;
    NormArgs p = {};
    p.x = x, p.r = r, p.h = h, p.y = y, p.w = y || mx ? w : nullptr;        // the sum alone reads no weights, whatever w is
    p.ldx = ld_x, p.ldr = ld_r, p.ldh = ld_h, p.ldy = ld_y;
    if (mx) p.o = mx_out(*mx);
    p.rows = n_tok, p.cols = cols;
    p.eps = eps;
    p.mean = 1.0 / cols;
    p.vec_in = on_16(x, ld_x, t) && (!r || on_16(r, ld_r, t)) && (uintptr_t)p.w % 16 == 0;
    p.vec_out = (!h || on_16(h, ld_h, t)) && (!y || on_16(y, ld_y, t));
    const int64_t size = (int64_t)lm_type_size(t);
    p.x_end = (const char *)x + ((n_tok - 1) * ld_x + cols) * size;
    p.r_end = (const char *)r + ((n_tok - 1) * ld_r + cols) * size;
    return lm_by_type(t, [&](auto v) { return norm_go<decltype(v)>(p); });
}
