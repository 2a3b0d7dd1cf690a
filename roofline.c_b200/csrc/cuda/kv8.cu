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
// write the same bytes; it reads its new rows twice, once for the largest
// magnitude and once (from L1/L2) for the codes. Bound by memory for prompts
// (4 or 2 bytes in, 1 out per element) and by the latency of four dependent
// loads (lengths, page, scale, row) for a decode step.
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

// This CTA's page: grid (sequence x page, head, K or V). False when there is
// nothing to do; page -1 when the table names none.
__device__ __forceinline__ bool place_of(const RowsArgs &p, kv8_place_t &at, int &page)
{
    const int b = blockIdx.x / p.reach, j = blockIdx.x % p.reach;
    const bool report = threadIdx.x == 0;
    kv8_seq_t q;
    if (!kv_seq(p.step, b, q, p.err, report) || !kv8_place(&q, j, &at)) return false;
    page = kv_page(p.step, b, at.index, p.n_pages, p.err, report);
    return true;
}

__device__ __forceinline__ int8_t code_of(float x, float s)
{
    // x finite; the clamp is for the quotients of a subnormal scale
    return s > 0.0f ? (int8_t)(int)fminf(fmaxf(rintf(__fdiv_rn(x, s)), -127.0f), 127.0f) : (int8_t)0;
}

// What is stored for a value: 0 for a NaN, the largest finite magnitude for an infinity.
__device__ __forceinline__ float finite(float x)
{
    return x == x ? fminf(fmaxf(x, -3.402823466e38f), 3.402823466e38f) : 0.0f;
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

template <typename T, int V>
__global__ void __launch_bounds__(256) append_kernel(const RowsArgs p)
{
    __shared__ float s_max[8];
    __shared__ __align__(16) uint8_t s_code[128 * 68];   // V: [dim][slot], rows of 68 bytes
    pdl_wait();
    kv8_place_t at;
    int page;
    if (!place_of(p, at, page) || page < 0) return;
    const int side = blockIdx.z, head = blockIdx.y, D = p.D, n = at.hi - at.lo, per = D / V;
    const T *x = (const T *)p.x[side] + at.row * p.ld[side] + (long long)head * D;
    const long long ld = p.ld[side], ph = (long long)page * p.n_kv + head;
    float *const scale = p.scale[side] + ph;
    const float was = at.lo ? *scale : 0.0f;

    float m = 0.0f;
    for (int i = threadIdx.x; i < n * per; i += blockDim.x) {
        float v[V];
        load_pack<T, V>(x + (i / per) * ld + (i % per) * V, v);
#pragma unroll
        for (int e = 0; e < V; e++) m = fmaxf(m, fabsf(finite(v[e])));
    }
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
    __syncthreads();                                     // also: `was` is read by all before it is replaced
    m = s_max[0];
    for (int i = 1; i < (int)blockDim.x / 32; i++) m = fmaxf(m, s_max[i]);
    const float now = fmaxf(was, __fdiv_rn(m, 127.0f));
    const float ratio = now > was && now > 0.0f ? __fdiv_rn(was, now) : 1.0f;
    if (threadIdx.x == 0) *scale = now;

    int8_t *const code = p.code[side] + ph * TCG_KV8_PAGE * D;
    const bool move = ratio != 1.0f && at.lo;
    if (side == 0) {                                     // K: token-major
        if (move) {
            uint32_t *w = (uint32_t *)code;
            for (int i = threadIdx.x; i < at.lo * D / 4; i += blockDim.x) w[i] = moved4(w[i], ratio);
        }
        for (int i = threadIdx.x; i < n * per; i += blockDim.x) {
            float v[V];
            load_pack<T, V>(x + (i / per) * ld + (i % per) * V, v);
            Pack<int8_t, V> c;
#pragma unroll
            for (int e = 0; e < V; e++) c.v[e] = code_of(finite(v[e]), now);
            *(Pack<int8_t, V> *)(code + (at.lo + i / per) * D + (i % per) * V) = c;
        }
        return;
    }
    // V: dim-major. The codes go to shared memory as [dim][slot]; then the words (4 slots) that hold a new token, or
    // an older one to move, are put together and written.
    for (int i = threadIdx.x; i < n * per; i += blockDim.x) {
        float v[V];
        load_pack<T, V>(x + (i / per) * ld + (i % per) * V, v);
#pragma unroll
        for (int e = 0; e < V; e++)
            s_code[((i % per) * V + e) * 68 + at.lo + i / per] =
                (uint8_t)code_of(finite(v[e]), now);
    }
    __syncthreads();
    const int w0 = move ? 0 : at.lo / 4, w1 = (at.hi + 3) / 4, nw = w1 - w0;
    uint32_t *const row = (uint32_t *)code;
    for (int i = threadIdx.x; i < D * nw; i += blockDim.x) {
        const int d = i / nw, w = w0 + i % nw;
        uint32_t *const dst = row + d * (TCG_KV8_PAGE / 4) + w;
        uint32_t fresh = 0;                              // bytes of the word that are new tokens
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (4 * w + e >= at.lo && 4 * w + e < at.hi) fresh |= 0xFFu << (8 * e);
        uint32_t v = 0;
        if (fresh) v = *(const uint32_t *)(s_code + d * 68 + 4 * w) & fresh;
        if (fresh != 0xFFFFFFFFu) {
            const uint32_t old = *dst;
            uint32_t keep = old;
            if (move) {
                const uint32_t mv = moved4(old, ratio);
                uint32_t older = 0;
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (4 * w + e < at.lo) older |= 0xFFu << (8 * e);
                keep = (mv & older) | (old & ~older);
            }
            v |= keep & ~fresh;
        }
        *dst = v;
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(256) read_kernel(const RowsArgs p)
{
    __shared__ __align__(16) uint8_t s_code[128 * 68];
    pdl_wait();
    kv8_place_t at;
    int page;
    if (!place_of(p, at, page)) return;
    const int side = blockIdx.z, head = blockIdx.y, D = p.D, n = at.hi - at.lo, per = D / V;
    T *y = (T *)p.y[side] + at.row * p.ld[side] + (long long)head * D;
    const bool bad = page < 0;
    const long long ld = p.ld[side], ph = (long long)(bad ? 0 : page) * p.n_kv + head;
    const float scale = bad ? 0.0f : p.scale[side][ph];
    const int8_t *const code = p.code[side] + ph * TCG_KV8_PAGE * D;
    if (side == 1) {
        const int w0 = at.lo / 4, nw = (at.hi + 3) / 4 - w0;
        const uint32_t *const row = (const uint32_t *)code;
        for (int i = threadIdx.x; i < D * nw; i += blockDim.x) {
            const int d = i / nw, w = w0 + i % nw;
            *(uint32_t *)(s_code + d * 68 + 4 * w) = row[d * (TCG_KV8_PAGE / 4) + w];
        }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < n * per; i += blockDim.x) {
        const int r = i / per, d = (i % per) * V;
        float v[V];
        if (side == 0) {
            const Pack<int8_t, V> c = *(const Pack<int8_t, V> *)(code + (at.lo + r) * D + d);
#pragma unroll
            for (int e = 0; e < V; e++) v[e] = (float)c.v[e];
        } else {
#pragma unroll
            for (int e = 0; e < V; e++) v[e] = (float)(int8_t)s_code[(d + e) * 68 + at.lo + r];
        }
#pragma unroll
        for (int e = 0; e < V; e++) v[e] = bad ? 0.0f : v[e] * scale;
        store_pack<T, V>(y + r * ld + d, v);
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
    p.err = ctx().d_err;
    const long long gx = (long long)s->n_seq * p.reach;
    if (gx > 0x7fffffffll) return fail("%s: %d sequences of up to %d tokens are too many for one call", who, s->n_seq, longest);
    const bool vec = ((uintptr_t)k | (uintptr_t)v) % (4 * size) == 0 && ld_k % 4 == 0 && ld_v % 4 == 0;
    const dim3 grid((unsigned)gx, (unsigned)c->n_kv_head, 2), block(longest >= 8 ? 256 : 64);
    return lm_by_type(t, [&](auto e) {
        using T = decltype(e);
        void (*fn)(const RowsArgs) = append ? (vec ? append_kernel<T, 4> : append_kernel<T, 1>)
                                            : (vec ? read_kernel<T, 4> : read_kernel<T, 1>);
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
