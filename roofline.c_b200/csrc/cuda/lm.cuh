// lm.cuh -- what the language-model operators (rope.cu, kv8.cu, kv8_attn.cu)
// share: the three activation types and their vector loads and stores, the
// checks of arguments, and the device-side reading of a step's lengths.
#pragma once

#include "kv8_index.h"
#include "tcg_common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace tcg {

// True (no message) when the library has a device and it is the current one:
// a launch on the library's stream from another device's context would fail.
inline bool lm_ready(const char *who)
{
    if (!need_ctx()) return false;
    int dev = -1;
    TCG_CUDA(cudaGetDevice(&dev));
    if (dev != ctx().device)
        return fail("%s: device %d is current, this thread's library device is %d", who, dev, ctx().device);
    return true;
}

// Their own device error word, apart from the one that makes a host-buffer op abort.
inline int *lm_error_word() { return ctx().d_err + 2; }

inline size_t lm_type_size(ggml_type_t t)
{
    return t == GGML_TYPE_F32 ? 4 : t == GGML_TYPE_F16 || t == GGML_TYPE_BF16 ? 2 : 0;
}

// Calls f with a value of the element type t stands for.
template <typename F>
inline auto lm_by_type(ggml_type_t t, F &&f)
{
    if (t == GGML_TYPE_F32) return f(float());
    if (t == GGML_TYPE_F16) return f(__half());
    return f(__nv_bfloat16());
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Wait for the kernels before this one (programmatic dependent launch), then
// let the next one be scheduled if this one is `brief`: where a short grid
// leaves SMs free, the next one's start overlaps its work (the next one waits
// in turn for this grid's completion before it reads anything). After a larger
// grid it comes as the CTAs retire, which keeps its own evenly spread.
constexpr unsigned LM_SMALL_GRID = 148;
__device__ __forceinline__ void lm_signal(bool brief = true)
{
    if (brief && gridDim.x * gridDim.y * gridDim.z <= LM_SMALL_GRID)
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void lm_begin(bool brief = true)
{
    pdl_wait();
    lm_signal(brief);
}

// V consecutive elements as one access of V * sizeof(T) bytes (at most 16).
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
    T v[V];
};
template <typename T, int V>
__device__ __forceinline__ void load_pack(const T *p, float (&x)[V])
{
    const Pack<T, V> k = *reinterpret_cast<const Pack<T, V> *>(p);
#pragma unroll
    for (int i = 0; i < V; i++) x[i] = to_f32(k.v[i]);
}
template <typename T, int V>
__device__ __forceinline__ void store_pack(T *p, const float (&x)[V])
{
    Pack<T, V> k;
#pragma unroll
    for (int i = 0; i < V; i++) k.v[i] = from_f32<T>(x[i]);
    *reinterpret_cast<Pack<T, V> *>(p) = k;
}

// The pages and lengths of a step, as the kernels take them.
struct KvStep {
    const int32_t *tok_start, *kv_len, *table;
    int table_ld, n_tok, max_new;
};

// Sequence b's rows and length; false (and the device error word) when they
// cannot be. `report`: whether this thread raises the error word.
__device__ __forceinline__ bool kv_seq(const KvStep &s, int b, kv8_seq_t &q, int *err, bool report)
{
    if (kv8_seq_ok(s.tok_start[b], s.tok_start[b + 1], s.kv_len[b], s.n_tok, s.max_new, s.table_ld, &q)) return true;
    if (report) atomicExch(err, TCG_ERR_KV8_LENGTHS);
    return false;
}

// Page `p` of sequence b, or -1 (and the device error word) when the table
// names one that does not exist.
__device__ __forceinline__ int kv_page(const KvStep &s, int b, int p, int n_pages, int *err, bool report)
{
    const int g = s.table[(size_t)b * s.table_ld + p];
    if (kv8_page_ok(g, n_pages)) return g;
    if (report) atomicExch(err, TCG_ERR_KV8_PAGE);
    return -1;
}

// Checks of a cache and a step that need no device.
bool kv8_check(const char *who, const tcg_kv8_t *c, const tcg_kv8_step_t *s, ggml_type_t t);

inline KvStep kv_step(const tcg_kv8_step_t &s)
{
    return { s.tok_start, s.kv_len, s.table, s.table_ld, s.n_tok, s.max_new };
}

}  // namespace tcg
