// kv8_attn.cuh -- what the two kernels of tcg_kv8_attention share: the
// arguments, reading query rows, writing output rows.
#pragma once

#include "lm.cuh"

#include <math.h>

#include <atomic>

namespace tcg {

constexpr int PAGE = TCG_KV8_PAGE;
constexpr int ERR_WAIT = TCG_ERR_KV8_WAIT;

struct AttnArgs {
    const void *q;
    void *out;
    long long ld_q, ld_out;
    int type, q_vec, out_vec;            // ggml type; 16-byte loads / 4-element stores possible
    const int8_t *v;
    const float *k_scale, *v_scale;
    KvStep step;
    int n_pages, n_kv, n_seq, D, G;
    unsigned g_inv, d4_inv;              // n / G and n / (D / 4) are n * inv >> 20 where n times the divisor is below 2^20
    float scale_log2;
    int causal, window;
    int ntile, S;                        // blocks of rows a sequence; CTAs (a cluster) that share one's keys
    int brief;                           // a few rounds of tiles at most
    int row_min;                         // only sequences of more than row_min rows (the kernel for many rows)
    int compact;                         // blocks of rows are dealt out by the lengths, not by (ntile, n_seq)
    int *err;
};

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// A score's factor without the values that would turn 0 or a masked -inf times it into NaN; a NaN (a query with a NaN or
// an infinity) stays.
__device__ __forceinline__ float tame(float c) { return c < 1e-37f ? 1e-37f : c > 3e38f ? 3e38f : c; }
// A scaled score within fp32's range, which differences of two of them pass to -inf only.
__device__ __forceinline__ float in_range(float x) { return fminf(fmaxf(x, -3e38f), 3e38f); }

// Scaled scores beyond this are subtracted before they are scaled: fp32's rounding of the product, 2^-24 of it, would
// otherwise enter the exponent (at 2^27 the row's largest weight came out as 2^-32).
constexpr float FAR_SCORE = 4096.0f;

// 16 consecutive values of a query row.
__device__ __forceinline__ void load_q16(const AttnArgs &p, long long off, float (&x)[16])
{
    if (p.type == GGML_TYPE_F32) {
        const float *s = (const float *)p.q + off;
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            if (p.q_vec) {
                const float4 v = *(const float4 *)(s + i);
                x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) x[i + e] = s[i + e];
            }
        }
        return;
    }
    const unsigned short *s = (const unsigned short *)p.q + off;
    uint32_t w[8];
    if (p.q_vec) {
        const uint4 a = *(const uint4 *)s, b = *(const uint4 *)(s + 8);
        w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = (uint32_t)s[2 * i] | (uint32_t)s[2 * i + 1] << 16;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        if (p.type == GGML_TYPE_BF16) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        } else {
            x[2 * i] = __half2float(__ushort_as_half((unsigned short)w[i]));
            x[2 * i + 1] = __half2float(__ushort_as_half((unsigned short)(w[i] >> 16)));
        }
    }
}

template <int V>
__device__ __forceinline__ void store_out(const AttnArgs &p, long long off, const float (&x)[V])
{
    if (p.type == GGML_TYPE_F32) {
        float *o = (float *)p.out + off;
        if (p.out_vec) store_pack<float, V>(o, x);
        else
#pragma unroll
            for (int i = 0; i < V; i++) o[i] = x[i];
    } else if (p.type == GGML_TYPE_F16) {
        __half *o = (__half *)p.out + off;
        if (p.out_vec) store_pack<__half, V>(o, x);
        else
#pragma unroll
            for (int i = 0; i < V; i++) o[i] = __float2half_rn(x[i]);
    } else {
        __nv_bfloat16 *o = (__nv_bfloat16 *)p.out + off;
        if (p.out_vec) store_pack<__nv_bfloat16, V>(o, x);
        else
#pragma unroll
            for (int i = 0; i < V; i++) o[i] = __float2bfloat16_rn(x[i]);
    }
}

// Sum of weights -> factor on O. A row that saw nothing has the sum 0 and
// gets zeros; a NaN sum (a query with a NaN or an infinity) stays NaN.
__device__ __forceinline__ float inverse(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }

__device__ __forceinline__ uint32_t mapa(uint32_t a, int rank)
{
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    return r;
}
__device__ __forceinline__ float ld_cluster(uint32_t a)
{
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a));
    return v;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t a)
{
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

constexpr int MAX_SPLIT = 10;            // CTAs of a cluster; of 11 or more a B200 holds 7 clusters at a time

// Four output values of a row from the S CTAs of a cluster: their maxima, sums and O's at these shared-memory addresses,
// read together (MAX at least S), joined in the CTAs' order, times `unit`.
template <int MAX>
__device__ __forceinline__ void cluster_join(uint32_t a_m, uint32_t a_l, uint32_t a_o, int S, float unit, float (&v)[4])
{
    float m[MAX], l[MAX], top = -INFINITY, sum = 0.0f;
    float4 x[MAX];
#pragma unroll
    for (int s = 0; s < MAX; s++) {
        m[s] = -INFINITY, l[s] = 0.0f, x[s] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (s < S) {
            m[s] = ld_cluster(mapa(a_m, s));
            l[s] = ld_cluster(mapa(a_l, s));
            x[s] = ld_cluster4(mapa(a_o, s));
        }
    }
#pragma unroll
    for (int s = 0; s < MAX; s++) top = fmaxf(top, m[s]);
    top = top == -INFINITY ? 0.0f : top;
    v[0] = v[1] = v[2] = v[3] = 0.0f;
#pragma unroll
    for (int s = 0; s < MAX; s++) {
        const float w = ex2(m[s] - top);
        sum = fmaf(w, l[s], sum);
        v[0] = fmaf(w, x[s].x, v[0]), v[1] = fmaf(w, x[s].y, v[1]), v[2] = fmaf(w, x[s].z, v[2]), v[3] = fmaf(w, x[s].w, v[3]);
    }
    const float inv = inverse(sum) * unit;
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] *= inv;
}


// Launches FN over ntile x n_seq x n_kv blocks of rows with `tiles` tiles of keys each at most, of which `groups` are
// taken at a time, after choosing the split of the keys over a cluster of S CTAs. rows: of a block; per_sm: CTAs an SM.
template <auto FN, typename X>
bool attn_grid(AttnArgs &p, dim3 block, size_t smem, int rows, int per_sm, long long tiles, int groups, const X &arg)
{
    cudaLaunchAttribute attrs[2];
    cudaLaunchConfig_t lc = {};
    lc.blockDim = block;
    lc.dynamicSmemBytes = smem;
    lc.stream = ctx().cur;
    lc.attrs = attrs;
    // SMs that clusters of a size can use at once (a property of the device: its SMs come in groups that a cluster does not
    // cross); the first call prepares the kernel, too. Threads that come first together write the same; sms[1] says that
    // the others are there.
    static std::atomic<int> usable[64][MAX_SPLIT + 1];
    std::atomic<int> *const sms = usable[ctx().device & 63];
    if (!sms[1].load(std::memory_order_acquire)) {
        TCG_CUDA(cudaFuncSetAttribute(FN, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        TCG_CUDA(cudaFuncSetAttribute(FN, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        attrs[0].id = cudaLaunchAttributeClusterDimension;
        attrs[0].val.clusterDim.y = attrs[0].val.clusterDim.z = 1;
        cudaLaunchConfig_t one = lc;
        one.numAttrs = 1;
        for (int S = MAX_SPLIT; S > 1; S--) {
            int n = 0;
            one.gridDim = dim3((unsigned)S);
            attrs[0].val.clusterDim.x = (unsigned)S;
            if (cudaOccupancyMaxActiveClusters(&n, FN, &one) != cudaSuccess) {
                cudaGetLastError();
                n = 0;
            }
            sms[S].store(n * S < ctx().sms ? n * S : ctx().sms, std::memory_order_relaxed);
        }
        sms[1].store(ctx().sms, std::memory_order_release);
    }
    // The split: the S with the least work for the busiest SM, in tiles: its CTAs' rounds of tiles and about two more each
    // (start, merge). A second CTA on the SM fills the first one's waits: two take 1.5 times as long as one, measured.
    const long long all = (long long)p.ntile * p.n_seq;
    const long long even = ((long long)p.step.n_tok * p.G + rows - 1) / rows, full = even + p.n_seq;   // with rows, at most
    p.compact = all > 2 * full + 64;                         // and one block more, which sees every sequence
    const long long ctas = (p.compact ? full + 1 : all) * p.n_kv, likely = p.row_min ? even + 1 : full;
    const long long busy = (all < likely ? all : likely) * p.n_kv;
    p.S = 1;
    long long best = 0, last = 0;
    for (int S = 1; S <= MAX_SPLIT; S++) {
        const int at_once = sms[S].load(std::memory_order_relaxed);
        if (!at_once || (S > 1 && tiles < (long long)S * groups) || (p.compact && S > 2)) continue;   // compact: most are empty
        const long long n = (busy * S + at_once - 1) / at_once;
        const long long rounds = ((tiles + S - 1) / S + groups - 1) / groups, t = n * (rounds + 2) * (n > 1 && per_sm > 1 ? 3 : 4);
        if (S == 1 || t < best) best = t, p.S = S, last = rounds;
    }
    p.brief = last <= 4;
    if (ctas * p.S > 0x7fffffffll)
        return fail("tcg_kv8_attention: %d sequences of %d row blocks and %d key heads are too many for one call", p.n_seq,
                    p.ntile, p.n_kv);
    lc.gridDim = dim3((unsigned)(ctas * p.S));
    lc.numAttrs = pdl_attr(attrs);
    if (p.S > 1) {
        attrs[lc.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attrs[lc.numAttrs].val.clusterDim.x = (unsigned)p.S;
        attrs[lc.numAttrs].val.clusterDim.y = 1;
        attrs[lc.numAttrs].val.clusterDim.z = 1;
        lc.numAttrs++;
    }
    TCG_CUDA(cudaLaunchKernelEx(&lc, FN, p, arg));
    return true;
}

// The kernel for many rows (kv8_attn_tc.cu): 128 rows a CTA on the 5th-generation
// tensor cores. R: the most rows a sequence has, tiles: pages of keys.
bool launch_kv8_attn_tc(AttnArgs &p, const int8_t *k, long long R, long long tiles);

}  // namespace tcg
