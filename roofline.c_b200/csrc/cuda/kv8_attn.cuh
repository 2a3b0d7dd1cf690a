// kv8_attn.cuh -- what the two kernels of tcg_kv8_attention share: the
// arguments, reading query rows, writing output rows.
#pragma once

#include "lm.cuh"

namespace tcg {

constexpr int PAGE = TCG_KV8_PAGE;
constexpr int ERR_WAIT = 66;             // device error word: a tile's copy did not land in time

struct AttnArgs {
    const void *q;
    void *out;
    long long ld_q, ld_out;
    int type, q_vec, out_vec;            // ggml type; 16-byte loads / 4-element stores possible
    const int8_t *v;
    const float *k_scale, *v_scale;
    KvStep step;
    int n_pages, n_kv, D, G;
    float scale_log2;
    int causal, window, S;
    int *err;
};

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
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

// The kernel for many rows (kv8_attn_tc.cu): 128 rows a CTA on the 5th-generation
// tensor cores.
bool launch_kv8_attn_tc(AttnArgs &p, const int8_t *k, long long R, int n_seq);

}  // namespace tcg
