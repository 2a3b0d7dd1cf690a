// kv8.cu -- the 8-bit key/value cache: writing a step's rows
// (tcg_kv8_append) and reading rows back (tcg_kv8_read).
//
// A page holds 64 tokens; a (page, head) has one fp32 scale for K and one for
// V, value = code * scale. Appending to a page with scale s (0 when the page
// starts with the new tokens) and largest new magnitude m:
//   s' = max(s, fl(m / 127)),  code = rint(fl(x / s')) in -127 .. 127,
//   older codes <- rint(fl(code * fl(s / s')))    when s' > s,
// each fl one rounding to fp32, so that the stored bytes are defined exactly.
// One CTA owns a (page, head, K or V) and everything in it, so no two CTAs
// write the same bytes; its new rows are read once, into registers. Bound by
// memory for prompts in principle (4 or 2 bytes in, 1 out per element); as it
// is, by instructions, about 22 a value: five f16 prompts up to 2048 tokens
// (8 heads of 128) 14 us, and 11 us to read them back as fp32. A decode step
// is bound by the latency of dependent loads (lengths, page, scale): 33 tokens
// 3.8 us, their pages read back 6.1 us, 8.7 us for both in a row (back to back;
// an empty kernel launched the same way 2.6 us).
#include "lm.cuh"

namespace tcg {

bool kv8_check(const char *who, const tcg_kv8_t *c, const tcg_kv8_step_t *s, ggml_type_t t)
{
    if (!c || !s) return fail("%s: no cache or no step", who);
    if (!lm_type_size(t)) return fail("%s: type %d is not F32, F16 or BF16", who, (int)t);
    if (c->head_dim < 16 || c->head_dim > 128 || c->head_dim % 16)
        return fail("%s: head_dim %d is not a multiple of 16 in 16 .. 128", who, c->head_dim);
    if (c->n_kv_head < 1 || c->n_kv_head > 65535) return fail("%s: %d key heads", who, c->n_kv_head);
    if (c->n_pages < 1 || (long long)c->n_pages * c->n_kv_head * TCG_KV8_PAGE > 0x7fffffffll)
        return fail("%s: %d pages of %d heads: pages x heads x 64 is not in 1 .. 2^31 - 1", who, c->n_pages, c->n_kv_head);
    if (!c->k || !c->v || !c->k_scale || !c->v_scale) return fail("%s: the cache has no memory", who);
    if (((uintptr_t)c->k | (uintptr_t)c->v) % 16 || ((uintptr_t)c->k_scale | (uintptr_t)c->v_scale) % 4)
        return fail("%s: the cache's codes are not 16-byte aligned, or its scales not 4-byte aligned", who);
    if (s->n_seq < 0 || s->n_seq > 65535 || s->n_tok < 0 || s->max_new < 0 || s->max_kv < 0 || s->table_ld < 0)
        return fail("%s: a count of the step is negative, or there are more than 65535 sequences", who);
    if (s->n_seq && (!s->tok_start || !s->kv_len || (!s->table && s->table_ld))) return fail("%s: the step has no arrays", who);
    if (((uintptr_t)s->tok_start | (uintptr_t)s->kv_len | (uintptr_t)s->table) % 4) return fail("%s: misaligned step arrays", who);
    return true;
}

namespace {

// Grid: (sequence x page that its rows touch, head, K or V).
struct RowsArgs {
    const void *x[2];             // new K rows, new V rows (append)
    void *y[2];                   // rows to fill (read)
    long long ld[2];
    int8_t *code[2];
    float *scale[2];
    KvStep step;
    int n_pages, n_kv, D, reach;  // pages that a sequence's rows can touch
    int *err;
};

// What is stored for a value: 0 for a NaN, the largest finite magnitude for an infinity.
__device__ __forceinline__ float finite(float x)
{
    return x == x ? fminf(fmaxf(x, -3.402823466e38f), 3.402823466e38f) : 0.0f;
}

// A product of a code and a scale, which rounds to an infinity for the largest ones (127 * fl(largest / 127)); NaN stays.
__device__ __forceinline__ float at_most_finite(float x)
{
    asm("min.NaN.xorsign.abs.f32 %0, %0, %1;" : "+f"(x) : "f"(3.402823466e38f));
    return x;
}

// The format's code for x at scale s, as it is defined. The clamp is for the quotients of a subnormal scale.
__device__ __forceinline__ int code_of(float x, float s)
{
    return s > 0.0f ? (int)fminf(fmaxf(rintf(__fdiv_rn(finite(x), s)), -127.0f), 127.0f) : 0;
}

// The same for N values of magnitude at most 127 s, as bytes in the low bits, with one product instead of a division:
// x * fl(1 / s) is within 127 * 2^-22 < 4e-5 of fl(x / s), so both round to the same whole number unless the product
// lies that near to a half (one value in 10,000); then the thread takes its values again by the definition. `plain`:
// every new value of the page is finite and s is at least 2^-100.
template <int N>
__device__ __forceinline__ void codes_of(const float (&x)[N], float s, float inv, bool plain, uint32_t (&c)[N])
{
    float off = plain ? 0.0f : 1.0f;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const float y = fmaf(x[i], inv, 12582912.0f);        // 1.5 * 2^23: the sum's low bits are the whole number
        off = fmaxf(off, fabsf(fmaf(x[i], inv, 12582912.0f - y)));
        c[i] = __float_as_uint(y);
    }
    if (off > 0.4999f) {
#pragma unroll
        for (int i = 0; i < N; i++) c[i] = (uint32_t)code_of(x[i], s);
    }
}

// The larger magnitude, NaN when either is.
__device__ __forceinline__ float max_nan(float m, float x)
{
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(m), "f"(fabsf(x)));
    return m;
}

// A code after its page's scale grew by 1 / ratio.
__device__ __forceinline__ int moved(int code, float ratio) { return (int)rintf(__fmul_rn((float)code, ratio)); }

__device__ __forceinline__ uint32_t moved4(uint32_t w, float ratio)
{
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) r |= (uint32_t)(moved((int8_t)(w >> (8 * i)), ratio) & 0xFF) << (8 * i);
    return r;
}

constexpr int ROWS_THREADS = 256;
constexpr int QUADS = TCG_KV8_PAGE / 4;      // groups of 4 slots
constexpr int S_PITCH = TCG_KV8_PAGE + 4;    // bytes of a dim's 64 codes in shared memory

// A thread owns V dims of 4 consecutive slots, up to 8 / V times (32 values):
// dims (thread % per) * V, quads thread / per, + `stride`, ..., per = D / V.
// Lanes run along a row, so rows are read and written whole; the 4 slots of a
// dim are one word of the dim-major V block.
template <int V>
struct Mine {
    static constexpr int N = 8 / V;
    int d, quad, stride;
    bool in;
    __device__ explicit Mine(int D)
    {
        const int per = D / V;
        stride = ROWS_THREADS / per;
        quad = threadIdx.x / per;
        d = threadIdx.x % per * V;
        in = quad < stride;
    }
};

template <typename T, int V>
__global__ void __launch_bounds__(ROWS_THREADS) append_kernel(const RowsArgs p)
{
    __shared__ float s_max[ROWS_THREADS / 32];
    __shared__ __align__(16) uint8_t s_code[128 * S_PITCH];
    lm_begin();
    kv8_place_t at;
    kv8_seq_t q;
    const int b = blockIdx.x / p.reach, side = blockIdx.z, head = blockIdx.y, D = p.D;
    if (!kv_seq(p.step, b, q, p.err, threadIdx.x == 0) || !kv8_place(&q, blockIdx.x % p.reach, &at)) return;

    const Mine<V> my(D);
    const T *x = (const T *)p.x[side] + (at.row - at.lo) * p.ld[side] + (long long)head * D + my.d;
    const long long ld = p.ld[side];
    Pack<T, V> raw[Mine<V>::N][4];
#pragma unroll
    for (int k = 0; k < Mine<V>::N; k++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int slot = 4 * (my.quad + k * my.stride) + j;
            raw[k][j] = Pack<T, V>{};
            if (my.in && slot >= at.lo && slot < at.hi) raw[k][j] = *(const Pack<T, V> *)(x + slot * ld);
        }
    const int page = kv_page(p.step, b, at.index, p.n_pages, p.err, threadIdx.x == 0);
    if (page < 0) return;
    const long long ph = (long long)page * p.n_kv + head;
    float *const scale = p.scale[side] + ph;
    const float was = at.lo ? *scale : 0.0f;

    float m = 0.0f;
#pragma unroll
    for (int k = 0; k < Mine<V>::N; k++)
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int e = 0; e < V; e++) m = max_nan(m, to_f32(raw[k][j].v[e]));
    auto reduce = [&]() {
        for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
        if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
        __syncthreads();                                 // also: `was` is read by all before it is replaced
#pragma unroll
        for (int i = 0; i < ROWS_THREADS / 32; i++) m = max_nan(m, s_max[i]);
    };
    reduce();
    bool plain = m <= 3.402823466e38f;                   // the same for the whole CTA
    if (!plain) {
        __syncthreads();
        m = 0.0f;
#pragma unroll
        for (int k = 0; k < Mine<V>::N; k++)
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int e = 0; e < V; e++) m = max_nan(m, finite(to_f32(raw[k][j].v[e])));
        reduce();
    }
    const float now = fmaxf(was, __fdiv_rn(m, 127.0f));
    const float ratio = now > was && now > 0.0f ? __fdiv_rn(was, now) : 1.0f;
    if (threadIdx.x == 0) *scale = now;
    plain = plain && now >= 0x1p-100f;
    const float inv = plain ? __fdiv_rn(1.0f, now) : 0.0f;

    int8_t *const code = p.code[side] + ph * TCG_KV8_PAGE * D;
    const bool move = ratio != 1.0f && at.lo;
    if (side == 0) {                                     // K: token-major
        if (move) {
            uint32_t *w = (uint32_t *)code;
            for (int i = threadIdx.x; i < at.lo * D / 4; i += ROWS_THREADS) w[i] = moved4(w[i], ratio);
        }
#pragma unroll
        for (int k = 0; k < Mine<V>::N; k++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int slot = 4 * (my.quad + k * my.stride) + j;
                if (!my.in || slot < at.lo || slot >= at.hi) continue;
                float v[V];
                uint32_t q[V];
                Pack<int8_t, V> c;
#pragma unroll
                for (int e = 0; e < V; e++) v[e] = to_f32(raw[k][j].v[e]);
                codes_of(v, now, inv, plain, q);
#pragma unroll
                for (int e = 0; e < V; e++) c.v[e] = (int8_t)q[e];
                *(Pack<int8_t, V> *)(code + slot * D + my.d) = c;
            }
        return;
    }
    // V: dim-major. The new codes go to shared memory as [dim][slot], a word of 4 slots at a time; then the 16-byte
    // pieces of a dim that are all new are written whole, and of the others the words that hold a new token, or an
    // older one to move.
#pragma unroll
    for (int k = 0; k < Mine<V>::N; k++) {
        const int quad = my.quad + k * my.stride;
        if (!my.in || quad >= QUADS || 4 * quad + 3 < at.lo || 4 * quad >= at.hi) continue;
#pragma unroll
        for (int e = 0; e < V; e++) {
            float v[4];
            uint32_t q[4];
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = to_f32(raw[k][j].v[e]);
            codes_of(v, now, inv, plain, q);
            *(uint32_t *)(s_code + (my.d + e) * S_PITCH + 4 * quad) =
                __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < D * 4; i += ROWS_THREADS) {
        const int d = i / 4, s0 = i % 4 * 16;
        const uint32_t *const src = (const uint32_t *)(s_code + d * S_PITCH + s0);
        uint32_t *const dst = (uint32_t *)(code + d * TCG_KV8_PAGE + s0);
        if (s0 >= at.lo && s0 + 16 <= at.hi) {
            *(uint4 *)dst = make_uint4(src[0], src[1], src[2], src[3]);
            continue;
        }
        for (int w = 0; w < 4; w++) {
            const int slot = s0 + 4 * w;
            uint32_t fresh = 0, older = 0;               // bytes that are new tokens, and older ones
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (slot + e >= at.lo && slot + e < at.hi) fresh |= 0xFFu << (8 * e);
                if (slot + e < at.lo) older |= 0xFFu << (8 * e);
            }
            if (!fresh && !(move && older)) continue;
            uint32_t v = fresh ? src[w] & fresh : 0;
            if (fresh != 0xFFFFFFFFu) {
                const uint32_t old = dst[w];
                v |= (move ? (moved4(old, ratio) & older) | (old & ~older) : old) & ~fresh;
            }
            dst[w] = v;
        }
    }
}

// The same for up to FEW new tokens a sequence (a decode step): one warp per (page, head, side), a lane for 4 dims, no
// shared memory and no barrier.
constexpr int FEW = 4, FEW_WARPS = 4;

template <typename T, bool VEC>
__global__ void __launch_bounds__(32 * FEW_WARPS) append_few_kernel(const RowsArgs p, unsigned tasks)
{
    const unsigned task = blockIdx.x * FEW_WARPS + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31, D = p.D, d = 4 * lane;
    lm_begin();
    if (task >= tasks) return;
    const int side = task & 1, head = (task >> 1) % p.n_kv, bj = (task >> 1) / p.n_kv, b = bj / p.reach;
    kv8_place_t at;
    kv8_seq_t q;
    if (!kv_seq(p.step, b, q, p.err, lane == 0) || !kv8_place(&q, bj % p.reach, &at)) return;
    const int n = at.hi - at.lo;                         // at most FEW: a sequence has no more rows
    const T *x = (const T *)p.x[side] + at.row * p.ld[side] + (long long)head * D + d;
    float v[FEW][4] = {};
#pragma unroll
    for (int i = 0; i < FEW; i++)
        if (i < n && d < D) {
            if (VEC) {
                load_pack<T, 4>(x + i * p.ld[side], v[i]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) v[i][e] = to_f32(x[i * p.ld[side] + e]);
            }
        }
    const int page = kv_page(p.step, b, at.index, p.n_pages, p.err, lane == 0);
    if (page < 0) return;
    const long long ph = (long long)page * p.n_kv + head;
    float *const scale = p.scale[side] + ph;
    const float was = at.lo ? *scale : 0.0f;
    float m = 0.0f, top = 0.0f;
#pragma unroll
    for (int i = 0; i < FEW; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            m = max_nan(m, v[i][e]);
            top = fmaxf(top, fabsf(finite(v[i][e])));
        }
    for (int o = 16; o > 0; o >>= 1) {
        m = max_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    }
    const float now = fmaxf(was, __fdiv_rn(top, 127.0f));
    const float ratio = now > was && now > 0.0f ? __fdiv_rn(was, now) : 1.0f;
    if (lane == 0) *scale = now;                         // read by the whole warp before the shuffles
    const bool plain = m <= 3.402823466e38f && now >= 0x1p-100f;
    const float inv = plain ? __fdiv_rn(1.0f, now) : 0.0f;
    int8_t *const code = p.code[side] + ph * TCG_KV8_PAGE * D;
    if (ratio != 1.0f && at.lo) {
        // older codes; in V's words those of the slots from lo on are kept
        uint32_t *const w = (uint32_t *)code;
        const int words = side == 0 ? at.lo * D / 4 : D * QUADS;
#pragma unroll 4
        for (int i = lane; i < words; i += 32) {
            const int over = side == 0 ? 0 : 4 * (i % QUADS) + 4 - at.lo;    // slots of the word that are not older
            if (over >= 4) continue;
            const uint32_t keep = over <= 0 ? 0 : 0xFFFFFFFFu << (8 * (4 - over));
            w[i] = (moved4(w[i], ratio) & ~keep) | (w[i] & keep);
        }
        __syncwarp();
    }
    if (d >= D) return;
#pragma unroll
    for (int i = 0; i < FEW; i++) {
        if (i >= n) break;
        uint32_t c[4];
        codes_of(v[i], now, inv, plain, c);
        if (side == 0) {
            *(uint32_t *)(code + (at.lo + i) * D + d) =
                __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) code[(d + e) * TCG_KV8_PAGE + at.lo + i] = (int8_t)c[e];
        }
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(ROWS_THREADS) read_kernel(const RowsArgs p)
{
    __shared__ __align__(16) uint8_t s_code[128 * S_PITCH];
    lm_begin();
    kv8_place_t at;
    kv8_seq_t q;
    const int b = blockIdx.x / p.reach, side = blockIdx.z, head = blockIdx.y, D = p.D;
    if (!kv_seq(p.step, b, q, p.err, threadIdx.x == 0) || !kv8_place(&q, blockIdx.x % p.reach, &at)) return;
    const int page = kv_page(p.step, b, at.index, p.n_pages, p.err, threadIdx.x == 0);

    const Mine<V> my(D);
    const bool bad = page < 0;
    T *y = (T *)p.y[side] + (at.row - at.lo) * p.ld[side] + (long long)head * D + my.d;
    const long long ld = p.ld[side], ph = (long long)(bad ? 0 : page) * p.n_kv + head;
    const float scale = p.scale[side][ph];
    const int8_t *const code = p.code[side] + ph * TCG_KV8_PAGE * D;
    uint32_t w[Mine<V>::N][V];                           // side V: 4 slots of a dim; side K: the bytes of 4 slots below
    Pack<int8_t, V> c[Mine<V>::N][4];
    if (side == 1) {
        for (int i = threadIdx.x; i < D * 4; i += ROWS_THREADS) {
            const int d = i / 4, s0 = i % 4 * 16;
            if (s0 + 16 <= at.lo || s0 >= at.hi) continue;
            const uint4 v = *(const uint4 *)(code + d * TCG_KV8_PAGE + s0);
            uint32_t *const dst = (uint32_t *)(s_code + d * S_PITCH + s0);
            dst[0] = v.x, dst[1] = v.y, dst[2] = v.z, dst[3] = v.w;
        }
        __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < Mine<V>::N; k++) {
        const int quad = my.quad + k * my.stride;
        const bool any = my.in && quad < QUADS && 4 * quad + 3 >= at.lo && 4 * quad < at.hi;
        if (side == 1) {
#pragma unroll
            for (int e = 0; e < V; e++) w[k][e] = any ? *(const uint32_t *)(s_code + (my.d + e) * S_PITCH + 4 * quad) : 0;
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int e = 0; e < V; e++) c[k][j].v[e] = (int8_t)(w[k][e] >> (8 * j));
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int slot = 4 * quad + j;
                c[k][j] = Pack<int8_t, V>{};
                if (any && slot >= at.lo && slot < at.hi) c[k][j] = *(const Pack<int8_t, V> *)(code + slot * D + my.d);
            }
        }
    }
#pragma unroll
    for (int k = 0; k < Mine<V>::N; k++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int slot = 4 * (my.quad + k * my.stride) + j;
            if (!my.in || slot < at.lo || slot >= at.hi) continue;
            float v[V];
#pragma unroll
            for (int e = 0; e < V; e++) v[e] = bad ? 0.0f : at_most_finite((float)c[k][j].v[e] * scale);
            store_pack<T, V>(y + slot * ld, v);
        }
}

bool rows_go(const char *who, const tcg_kv8_t *c, const tcg_kv8_step_t *s, const void *k, const void *v, bool append,
             int64_t ld_k, int64_t ld_v, ggml_type_t t)
{
    if (!kv8_check(who, c, s, t)) return false;
    const size_t size = lm_type_size(t);
    const int64_t wide = (int64_t)c->n_kv_head * c->head_dim;
    if (s->n_tok && (!k || !v)) return fail("%s: no rows", who);
    if (((uintptr_t)k | (uintptr_t)v) % size) return fail("%s: misaligned rows", who);
    if ((ld_k < wide || ld_v < wide) && s->n_tok > 1)
        return fail("%s: rows of %lld values do not fit strides of %lld and %lld", who, (long long)wide, (long long)ld_k,
                    (long long)ld_v);
    if (!lm_ready(who)) return false;
    if (s->n_seq == 0 || s->n_tok == 0) return true;
    RowsArgs p = {};
    p.x[0] = k, p.x[1] = v;
    p.y[0] = (void *)k, p.y[1] = (void *)v;
    p.ld[0] = ld_k, p.ld[1] = ld_v;
    p.code[0] = c->k, p.code[1] = c->v;
    p.scale[0] = c->k_scale, p.scale[1] = c->v_scale;
    p.step = kv_step(*s);
    p.n_pages = c->n_pages, p.n_kv = c->n_kv_head, p.D = c->head_dim;
    const int longest = s->max_new < s->n_tok ? s->max_new : s->n_tok;
    p.reach = kv8_reach(longest);
    p.err = lm_error_word();
    const long long gx = (long long)s->n_seq * p.reach;
    if (gx > 0x7fffffffll) return fail("%s: %d sequences of up to %d tokens are too many for one call", who, s->n_seq, longest);
    const dim3 grid((unsigned)gx, (unsigned)c->n_kv_head, 2), block(ROWS_THREADS);
    return lm_by_type(t, [&](auto e) {
        using T = decltype(e);
        if (append && longest <= FEW && gx * c->n_kv_head * 2 <= 0x7fffffffll) {
            const unsigned tasks = (unsigned)(gx * c->n_kv_head * 2);
            const bool four = ((uintptr_t)k | (uintptr_t)v) % (4 * sizeof(T)) == 0 && ld_k % 4 == 0 && ld_v % 4 == 0;
            TCG_CUDA(launch_pdl(four ? append_few_kernel<T, true> : append_few_kernel<T, false>, dim3((tasks + FEW_WARPS - 1) / FEW_WARPS),
                                dim3(32 * FEW_WARPS), 0, ctx().cur, p, tasks));
            return true;
        }
        constexpr int W = 16 / sizeof(T);                // 16-byte packs where rows and pointers allow, else single values
        const bool vec = ((uintptr_t)k | (uintptr_t)v) % 16 == 0 && ld_k % W == 0 && ld_v % W == 0;
        void (*fn)(const RowsArgs) = append ? (vec ? append_kernel<T, W> : append_kernel<T, 1>)
                                            : (vec ? read_kernel<T, W> : read_kernel<T, 1>);
        TCG_CUDA(launch_pdl(fn, grid, block, 0, ctx().cur, p));
        return true;
    });
}

}  // namespace
}  // namespace tcg

using namespace tcg;

extern "C" bool tcg_kv8_append(const tcg_kv8_t *c, const tcg_kv8_step_t *s, const void *k, const void *v, int64_t ld_k,
                               int64_t ld_v, ggml_type_t t)
{
    return rows_go("tcg_kv8_append", c, s, k, v, true, ld_k, ld_v, t);
}

extern "C" bool tcg_kv8_read(void *k, void *v, const tcg_kv8_t *c, const tcg_kv8_step_t *s, int64_t ld_k, int64_t ld_v,
                             ggml_type_t t)
{
    return rows_go("tcg_kv8_read", c, s, k, v, false, ld_k, ld_v, t);
}
