// rope.cu -- rotary positions (tcg_rope), and the root-mean-square norm of
// every query and key head with the rotation in the same pass
// (tcg_qk_norm_rope).
//
// Pair i of a head at position p turns by the angle 2 pi p turns[i]:
//   (a, b) -> m (a cos - b sin, a sin + b cos).
// p * turns[i] is taken in 64 bits, its nearest whole number subtracted (the
// fraction of a revolution is then good to 2^-53 p turns, where a 32-bit
// angle at p = 2^20 would be off by 2^-4 radians), and only the fraction goes
// to fp32: sincospi(2 f). The norm is y = x / sqrt(mean(x^2) + eps) * w, its
// sum of squares in fp32 over the lanes of a head.
//
// Bound by memory: 2 * 4 bytes an element (fp32) for ~10 operations (4096 rows
// of 40 heads of 128 with norms, fp32: 30.3 us, 5.5 TB/s; 6001 rows of 36
// heads, half of each rotated, bf16: 23.3 us, 4.7 TB/s). A lane
// owns one "unit" of 2 V dims of a head, two vectors of V: V pairs of the
// rotated part, or 2 V dims of the rest. The warp computes its token's sines
// and cosines once, one pair a lane, and applies them to the heads of the
// token one after the other. 32 / L heads side by side in a
// warp, L = the lanes a head needs.
#include "lm.cuh"

namespace tcg {
namespace {

constexpr int ROPE_WARPS = 4;

// How a warp keeps loads in flight, by the element's size. 16-bit rows: one
// head's loads while the head before it is computed, and a token's heads dealt
// out until there are 64 warps an SM (6001 rows of 36 heads of 128 in bf16:
// 23.5 us; two heads at a time without that overlap 28.5, 16 warps 25.2).
// fp32 rows: two heads' loads at a time, 16 warps an SM (4096 rows of 40 heads
// with norms: 30.0 us; overlapped 32.3 to 41, 64 warps 35.3).
template <typename T>
struct Flow {
    static constexpr bool PIPE = sizeof(T) == 2;
    static constexpr int AHEAD = PIPE ? 1 : 2, WARPS_PER_SM = PIPE ? 64 : 16, CTAS = PIPE ? 8 : 6;
};

struct RopeArgs {
    const void *x[2];            // q (or the only tensor), k
    void *y[2];
    const float *w[2];           // norm weights
    long long ldx[2], ldy[2];
    const int32_t *pos;
    int heads[2];
    int n_tok, splits;           // a token's heads are dealt out to `splits` warps
    int D, n_rot, lanes;         // lanes of a head: a power of two, 1 .. 32
    float mscale, eps;
    double turns[TCG_ROPE_MAX_DIM / 2];
};

// The two vectors of unit u start at dims a and b. Pairs of the half layout
// and the dims that are not rotated come from two halves, each read by
// consecutive lanes without gaps.
template <int V, bool HALF>
__device__ __forceinline__ void unit_dims(int u, int n_rot, int D, int &a, int &b)
{
    const int half = n_rot / 2;
    if (u * V >= half) {
        a = n_rot + u * V - half;
        b = a + (D - n_rot) / 2;
    } else if (HALF) {
        a = u * V;
        b = a + half;
    } else {
        a = 2 * V * u;
        b = a + V;
    }
}

template <typename T, int V, int U, bool HALF, bool NORM>
__global__ void __launch_bounds__(32 * ROPE_WARPS, Flow<T>::CTAS) rope_kernel(const __grid_constant__ RopeArgs p)
{
    __shared__ __align__(16) float2 s_ang[ROPE_WARPS][TCG_ROPE_MAX_DIM / 2];
    constexpr int ROPE_AHEAD = Flow<T>::AHEAD;
    constexpr bool PIPE = Flow<T>::PIPE;
    const int lane = threadIdx.x & 31, L = p.lanes;
    const int sub = lane / L, l = lane % L, side = 32 / L;
    const unsigned task = blockIdx.x * ROPE_WARPS + (threadIdx.x >> 5);
    const int tok = (int)(task / p.splits), part = (int)(task % p.splits);
    const int units = p.D / (2 * V), all = p.heads[0] + p.heads[1], step = side * p.splits;

    int da[U], db[U];
    bool live[U], turn[U];
#pragma unroll
    for (int k = 0; k < U; k++) {
        const int u = l + 32 * k;
        live[k] = u < units;
        unit_dims<V, HALF>(live[k] ? u : 0, p.n_rot, p.D, da[k], db[k]);
        turn[k] = live[k] && u * V < p.n_rot / 2;
    }
    lm_begin();
    if (tok >= p.n_tok) return;

    // Batches of ROPE_AHEAD heads, whose loads go out together: the first before the angles are computed, with PIPE each
    // before the batch ahead of it is.
    struct Batch {
        Pack<T, V> a[ROPE_AHEAD][U], b[ROPE_AHEAD][U];
    };
    auto load = [&](Batch &x, int h0) {
#pragma unroll
        for (int j = 0; j < ROPE_AHEAD; j++) {
            const int h = h0 + j * step, s = h >= p.heads[0];
            const T *row = (const T *)p.x[s] + tok * p.ldx[s] + (h - (s ? p.heads[0] : 0)) * p.D;
#pragma unroll
            for (int k = 0; k < U; k++) {
                x.a[j][k] = x.b[j][k] = Pack<T, V>{};
                if (h < all && live[k]) {
                    x.a[j][k] = *(const Pack<T, V> *)(row + da[k]);
                    x.b[j][k] = *(const Pack<T, V> *)(row + db[k]);
                }
            }
        }
    };
    const int h_first = part * side + sub;
    Batch now, next;
    load(now, h_first);

    // The token's sines and cosines, a pair a lane, shared by the warp.
    const double at = (double)p.pos[tok];
    float2 *const ang = s_ang[threadIdx.x >> 5];
    for (int i = lane; i < p.n_rot / 2; i += 32) {
        const double t = at * p.turns[i];
        float2 a;
        sincospif((float)(2.0 * (t - rint(t))), &a.y, &a.x);
        ang[i] = make_float2(a.x * p.mscale, a.y * p.mscale);
    }
    __syncwarp();
    float cs[U][V], sn[U][V];
#pragma unroll
    for (int k = 0; k < U; k++)
#pragma unroll
        for (int i = 0; i < V; i++) {
            const float2 a = turn[k] ? ang[(l + 32 * k) * V + i] : make_float2(1.0f, 0.0f);
            cs[k][i] = a.x;
            sn[k][i] = a.y;
        }

    float w[U][2 * V];
    int have = -1;                                               // the side whose weights these are
    for (int h0 = h_first; h0 - sub < all; h0 += step * ROPE_AHEAD) {   // the warp's lanes leave together
        if (PIPE) load(next, h0 + step * ROPE_AHEAD);
        else if (h0 != h_first) load(now, h0);
#pragma unroll
        for (int j = 0; j < ROPE_AHEAD; j++) {
            const int h = h0 + j * step;
            if (h - sub >= all) break;                           // no lane of the warp has a head
            const int s = h >= p.heads[0];
            float v[U][2 * V], inv = 1.0f;
#pragma unroll
            for (int k = 0; k < U; k++)
#pragma unroll
                for (int i = 0; i < V; i++) {
                    v[k][i] = to_f32(now.a[j][k].v[i]);
                    v[k][V + i] = to_f32(now.b[j][k].v[i]);
                }
            if (NORM) {
                float ss = 0.0f;
#pragma unroll
                for (int k = 0; k < U; k++)
#pragma unroll
                    for (int i = 0; i < 2 * V; i++) ss = fmaf(v[k][i], v[k][i], ss);
                for (int o = L >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
                inv = rsqrtf(ss / (float)p.D + p.eps);
            }
            if (h >= all) continue;
            if (NORM && s != have) {
                have = s;
#pragma unroll
                for (int k = 0; k < U; k++)
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        w[k][i] = p.w[s][da[k] + i];
                        w[k][V + i] = p.w[s][db[k] + i];
                    }
            }
            T *row = (T *)p.y[s] + tok * p.ldy[s] + (h - (s ? p.heads[0] : 0)) * p.D;
#pragma unroll
            for (int k = 0; k < U; k++) {
                if (!live[k]) continue;
                float a[V], b[V];
                if (NORM) {
#pragma unroll
                    for (int i = 0; i < 2 * V; i++) v[k][i] = v[k][i] * inv * w[k][i];
                }
#pragma unroll
                for (int i = 0; i < V; i++) {
                    // the two values of pair i: one of each vector, or neighbours
                    float &lo = HALF ? v[k][i] : v[k][2 * i], &hi = HALF ? v[k][V + i] : v[k][2 * i + 1];
                    const float c = cs[k][i], d = sn[k][i], x = fmaf(lo, c, -(hi * d)), y = fmaf(lo, d, hi * c);
                    lo = turn[k] ? x : lo;
                    hi = turn[k] ? y : hi;
                }
#pragma unroll
                for (int i = 0; i < V; i++) {
                    a[i] = v[k][i];
                    b[i] = v[k][V + i];
                }
                store_pack<T, V>(row + da[k], a);
                store_pack<T, V>(row + db[k], b);
            }
        }
        if (PIPE) now = next;
    }
}

template <typename T, int V, int U>
bool rope_launch_v(const RopeArgs &p, bool half, bool norm, unsigned grid)
{
    void (*fn)(const RopeArgs) = half ? (norm ? rope_kernel<T, V, U, true, true> : rope_kernel<T, V, U, true, false>)
                                      : (norm ? rope_kernel<T, V, U, false, true> : rope_kernel<T, V, U, false, false>);
    TCG_CUDA(launch_pdl(fn, dim3(grid), dim3(32 * ROPE_WARPS), 0, ctx().cur, p));
    return true;
}

// Whether every vector of V elements of T starts at a multiple of its size:
// the units split both the rotated part and the rest, and rows and pointers
// are aligned.
template <typename T>
bool fits(const RopeArgs &p, bool half, int V)
{
    if (p.D % (2 * V) || (half ? p.n_rot / 2 % V || (p.D - p.n_rot) % (2 * V) : p.n_rot % (2 * V))) return false;
    for (int s = 0; s < 2; s++) {
        if (!p.heads[s]) continue;
        if (((uintptr_t)p.x[s] | (uintptr_t)p.y[s]) % (V * sizeof(T)) || p.ldx[s] % V || p.ldy[s] % V) return false;
    }
    return true;
}

template <typename T>
bool rope_launch(RopeArgs &p, bool half, bool norm)
{
    const int V = sizeof(T) == 2 && fits<T>(p, half, 8) ? 8 : fits<T>(p, half, 4) ? 4 : 1;
    const int units = p.D / (2 * V);
    p.lanes = 1;
    while (p.lanes < units && p.lanes < 32) p.lanes <<= 1;
    // A warp that takes all heads of its token computes the angles once; one
    // token or a few are dealt out to more warps, down to one head a lane
    // group, until there are enough warps an SM.
    const int side = 32 / p.lanes, all = p.heads[0] + p.heads[1], most = (all + side - 1) / side;
    long long want = ((long long)ctx().sms * Flow<T>::WARPS_PER_SM + p.n_tok - 1) / p.n_tok;
    p.splits = (int)(want < 1 ? 1 : want > most ? most : want);
    const long long warps = (long long)p.n_tok * p.splits;
    const long long grid = (warps + ROPE_WARPS - 1) / ROPE_WARPS;
    if (warps > 0x7fffffffll) return fail("rope: %d tokens of %d heads are too many for one call", p.n_tok, all);
    if constexpr (sizeof(T) == 2)
        if (V == 8) return rope_launch_v<T, 8, 1>(p, half, norm, (unsigned)grid);
    if (V == 4) return rope_launch_v<T, 4, 1>(p, half, norm, (unsigned)grid);
    if (units <= 32) return rope_launch_v<T, 1, 1>(p, half, norm, (unsigned)grid);
    return rope_launch_v<T, 1, TCG_ROPE_MAX_DIM / 64>(p, half, norm, (unsigned)grid);
}

bool rope_checks(const char *who, const tcg_rope_t *r, const int32_t *pos, int n_tok, ggml_type_t t)
{
    if (!lm_type_size(t)) return fail("%s: type %d is not F32, F16 or BF16", who, (int)t);
    if (!r || r->head_dim < 2 || r->head_dim > TCG_ROPE_MAX_DIM || (r->head_dim & 1) || r->n_rot < 2 ||
        r->n_rot > r->head_dim || (r->n_rot & 1) || (r->layout != TCG_ROPE_INTERLEAVED && r->layout != TCG_ROPE_HALF))
        return fail("%s: the plan is not initialised (tcg_rope_init)", who);
    if (n_tok < 0) return fail("%s: %d tokens", who, n_tok);
    if (n_tok && !pos) return fail("%s: no positions", who);
    return true;
}

bool rope_side(const char *who, const char *name, RopeArgs &p, int s, void *y, const void *x, const float *w, bool norm,
               int heads, int D, int64_t ldy, int64_t ldx, ggml_type_t t)
{
    p.heads[s] = heads;
    if (!heads) return true;
    if (!y || !x || (norm && !w)) return fail("%s: no %s, its output or its weights", who, name);
    if (((uintptr_t)y | (uintptr_t)x) % lm_type_size(t) || (uintptr_t)w % 4) return fail("%s: misaligned %s", who, name);
    if ((ldy < (int64_t)heads * D || ldx < (int64_t)heads * D) && p.n_tok > 1)
        return fail("%s: %s rows of %d heads of %d do not fit strides of %lld and %lld elements", who, name, heads, D,
                    (long long)ldx, (long long)ldy);
    p.x[s] = x;
    p.y[s] = y;
    p.w[s] = w;
    p.ldx[s] = ldx;
    p.ldy[s] = ldy;
    return true;
}

bool rope_go(const char *who, RopeArgs &p, const tcg_rope_t *r, const int32_t *pos, ggml_type_t t, bool norm)
{
    if (!lm_ready(who)) return false;
    if (p.n_tok == 0 || p.heads[0] + p.heads[1] == 0) return true;
    p.pos = pos;
    p.D = r->head_dim;
    p.n_rot = r->n_rot;
    p.mscale = r->mscale;
    for (int i = 0; i < r->n_rot / 2; i++) p.turns[i] = r->turns[i];
    return lm_by_type(t, [&](auto v) { return rope_launch<decltype(v)>(p, r->layout == TCG_ROPE_HALF, norm); });
}

}  // namespace
}  // namespace tcg

using namespace tcg;

extern "C" bool tcg_rope(void *out, const void *x, const int32_t *pos, const tcg_rope_t *r, int n_tok, int n_head,
                         int64_t ld_out, int64_t ld_x, ggml_type_t t)
{
    const char *who = "tcg_rope";
    if (!rope_checks(who, r, pos, n_tok, t)) return false;
    if (n_head < 0 || n_head > (1 << 20)) return fail("%s: %d heads", who, n_head);
    RopeArgs p = {};
    p.n_tok = n_tok;
    if (n_tok && !rope_side(who, "x", p, 0, out, x, nullptr, false, n_head, r->head_dim, ld_out, ld_x, t)) return false;
    return rope_go(who, p, r, pos, t, false);
}

extern "C" bool tcg_qk_norm_rope(void *q_out, void *k_out, const void *q, const void *k, const float *q_w,
                                 const float *k_w, float eps, const int32_t *pos, const tcg_rope_t *r, int n_tok,
                                 int n_head, int n_kv_head, int64_t ld_q_out, int64_t ld_k_out, int64_t ld_q,
                                 int64_t ld_k, ggml_type_t t)
{
    const char *who = "tcg_qk_norm_rope";
    if (!rope_checks(who, r, pos, n_tok, t)) return false;
    if (n_head < 0 || n_kv_head < 0 || n_head > (1 << 20) || n_kv_head > (1 << 20))
        return fail("%s: %d and %d heads", who, n_head, n_kv_head);
    if (!(eps >= 0.0f) || eps > 1e30f) return fail("%s: eps %g", who, (double)eps);
    RopeArgs p = {};
    p.n_tok = n_tok;
    p.eps = eps;
    if (n_tok && (!rope_side(who, "q", p, 0, q_out, q, q_w, true, n_head, r->head_dim, ld_q_out, ld_q, t) ||
                  !rope_side(who, "k", p, 1, k_out, k, k_w, true, n_kv_head, r->head_dim, ld_k_out, ld_k, t)))
        return false;
    return rope_go(who, p, r, pos, t, true);
}
