// kv8_attn_tc.cu -- tcg_kv8_attention for many rows (prompts and chunks of
// prompts) on the 5th-generation tensor cores.
//
// One CTA of 256 threads takes 128 consecutive query rows (row = token * G +
// query head of the group) of one key head; threads r and r + 128 share row r
// = TMEM lane r. A tile is two pages, 128 keys: thread r takes the first
// page's, r + 128 the second's, and half of the output dims each. A page's
// int8 K [64, D] and V [D, 64] are loaded into registers ahead of use,
// converted to fp16 (whole numbers up to 127: exact) and written to shared
// memory in the K-major, 128-byte-swizzled layout the MMA reads; V is
// dim-major in the cache, so neither is transposed. Then
//   S = Q K^T    128 x 128 fp32 in TMEM, Q as fp16 in shared memory;
//   softmax      x = S cs - m_g, cs = scale log2(e) 2^-e sk, P = exp2(x + 8);
//   P V          128 x D fp32 in TMEM, P as fp16 in TMEM over S's columns,
//                accumulated there over a group of tiles;
//   O = (O + sv0 2^(m_g - 8 - m) P V) 2^(m - m_new) at a group's end.
// Within a group the reference m_g and the V scale sv0 stay: a page's sv enters
// as log2(sv / sv0) in the exponent. m_g is the row's running maximum m, or 2^4
// over the maximum of the group's first tile where that is more than 2^8 below
// m (2^4, so that groups last: at the maximum itself, prompts of peaked scores
// take 5% longer). A group ends where a row's maximum outgrows its reference by
// 2^7, where sv and sv0 are 2^3 apart (a V of zeros is far from any), or after
// 4 tiles with fp32 inputs (32 otherwise): the tensor core's accumulation
// truncates, by about 2e-8 of the result per MMA, 64 (256) of them a group. A
// tile whose two pages' scales are 2^3 apart is taken twice, once
// for each page. So a weight is rounded (to 11 or 22 bits, or 2^-33 of 2^m_g)
// against weights of its own group, times V of about its own size: neither a
// key elsewhere that holds most of the weight nor a page of large V beside it
// takes its bits.
// O is used at a group's end only and lives in local memory.
// Q is scaled by a power of two per row into [2^14, 2^15). With fp16 or bf16
// inputs it is exact as one fp16, and P's rounding to fp16 (2^-11 of itself) is
// that of an fp16 output and below bf16's (over 2000 keys an fp16 result is off
// by 2.4e-4 to 2.9e-4, 2.1e-4 by its own rounding alone); with fp32 inputs Q
// and P are two fp16 pieces of 11 bits each (NP = 2), the small piece's
// products first.
//
// Why fp16 and not the 8-bit integers of the cache, as the kernel for few rows
// does: with one thread a row the integer path is bound by the threads' work
// on the accumulators (a conversion and a multiply-add for every digit of
// every value), which fp32 accumulators do not need; the conversion of K and V
// is shared by 128 rows.
//
// K and V of a tile take turns in one buffer (S is done with K before V is
// needed), so two CTAs fit an SM (with 256 TMEM columns each): the one's
// products run while the other's threads compute. Every wait is bounded as in
// attn_tc.cu.
//
// Measured, 32 query and 8 key heads: a 4096-token causal prompt 406 us fp32
// and 276 us bf16 with D = 128 (339 and 499 TFLOP/s), 4096 x 4096 without a
// mask 731 and 510 us (376 and 539 TFLOP/s), 512 tokens over 16384 with the
// keys split over clusters of 2 379 and 254 us. The tensor pipe is busy 33% of
// the time (fp32): the threads' own chain per tile is the limit. Four threads
// a row (64 registers) spill: 616 us. O in registers, folded every tile: 883
// us; 64-key tiles with a second S buffer: 497 us. (The last three when the
// kernel took 438 us.)
#include "kv8_attn.cuh"
#include "numerics.cuh"
#include "tc05.cuh"

#include <math.h>

#include <type_traits>

namespace tcg {
namespace {

constexpr int TC_THREADS = 256;
constexpr int TC_ROWS = 128;
constexpr uint32_t TC_COLS = 256;                // S, and P over it: 0 .. 127; P V: from 128
constexpr uint32_t Q_TILE = 128 * 128;           // [128 rows or keys x 64 fp16]
constexpr float P_BIAS = 8.0f, GROWTH = 7.0f;    // weights are up to 2^8, and 2^15 before a group ends (fp16: below 2^16)
constexpr float FAR_M = 8.0f, ROOM = 4.0f;       // a first maximum this far (log2) below m gets a reference of its own, ROOM above it
constexpr float NEAR_V = 3.0f;                   // log2 of how far a group's V scales are apart at most

template <int DP, int NP>
struct TcShape {
    static constexpr uint32_t Q = 0, KV = NP * (DP / 64) * Q_TILE, END = KV + (DP / 64) * Q_TILE;   // K, or V of 2 pages
    static constexpr uint32_t V_TILE = DP * 128;             // [DP dims x 64 keys]
    static constexpr size_t SMEM = 1024 + END + 32 + TC_THREADS * 4 * 2;
};

// D fp32, A and B fp16, both K-major, M = 128.
__device__ __forceinline__ constexpr uint32_t idesc_f16(int N)
{
    return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((128u >> 4) << 24);
}

// A from TMEM (row i in lane i, two fp16 of K per column), B from shared memory.
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a_tmem, unsigned long long b, uint32_t id, uint32_t acc)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a_tmem), "l"(b), "r"(id), "r"(acc));
}

// 16 columns of this thread's TMEM lane from registers; waits for the store.
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0],"
                 " {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n\t"
                 "tcgen05.wait::st.sync.aligned;"
                 ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]),
                   "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]),
                   "r"(v[15])
                 : "memory");
}

// Byte offset of 16-byte chunk c of row r of a swizzled tile with rows of 128 bytes.
__device__ __forceinline__ uint32_t chunk_at(int r, int c) { return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)); }

// 16 codes as fp16, the two 16-byte chunks c and c + 1 of row r. A byte u =
// code + 128 under the exponent byte 0x64 is the fp16 number 1024 + u.
__device__ __forceinline__ void store_codes(uint8_t *tile, int r, int c, uint4 raw)
{
    const uint32_t w[4] = { raw.x, raw.y, raw.z, raw.w };
    uint32_t h[8];
    const __half2 off = __float2half2_rn(1152.0f);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t u = w[i] ^ 0x80808080u;
        const uint32_t lo = __byte_perm(u, 0x64646464u, 0x4140), hi = __byte_perm(u, 0x64646464u, 0x4342);
        const __half2 a = __hsub2(*(const __half2 *)&lo, off), b = __hsub2(*(const __half2 *)&hi, off);
        h[2 * i] = *(const uint32_t *)&a;
        h[2 * i + 1] = *(const uint32_t *)&b;
    }
    *(uint4 *)(tile + chunk_at(r, c)) = make_uint4(h[0], h[1], h[2], h[3]);
    *(uint4 *)(tile + chunk_at(r, c + 1)) = make_uint4(h[4], h[5], h[6], h[7]);
}

// The block of rows that number `want` over all sequences with rows in this launch stands for, found by a warp
// from the lengths; false behind the last one. For batches of unlike lengths (one prompt among decode steps), where a
// grid of ntile x n_seq would be nearly empty. A warp that finds none has seen, and reported, every sequence.
__device__ __forceinline__ bool find_block(const AttnArgs &p, int want, int &b, int &block)
{
    constexpr int SETS = 4;                                  // of 32 sequences, whose lengths are asked for together
    const int lane = threadIdx.x & 31;
    int before = 0;
    for (int s0 = 0; s0 < p.n_seq; s0 += 32 * SETS) {
        int n[SETS];
#pragma unroll
        for (int k = 0; k < SETS; k++) {
            const int s = s0 + 32 * k + lane;
            kv8_seq_t q;
            n[k] = 0;
            if (s < p.n_seq && kv_seq(p.step, s, q, p.err, true)) {
                const int R = q.n * p.G;
                if (R > p.row_min) n[k] = (R + TC_ROWS - 1) / TC_ROWS;
            }
        }
#pragma unroll
        for (int k = 0; k < SETS; k++) {
            int upto = n[k];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
                if (lane >= o) upto += v;
            }
            const unsigned past = __ballot_sync(0xFFFFFFFFu, before + upto > want);
            if (past) {
                const int l = __ffs((int)past) - 1;
                b = s0 + 32 * k + l;
                block = want - before - __shfl_sync(0xFFFFFFFFu, upto - n[k], l);
                return true;
            }
            before += __shfl_sync(0xFFFFFFFFu, upto, 31);
        }
    }
    return false;
}

// This CTA's sequence, block of rows, key head and rank in its cluster; `shared`: two words that nothing else uses. Grid:
// (rows from the last, sequence, head, rank), so that the blocks with the most keys start first. False, for the whole CTA
// and cluster, where there is none.
__device__ __forceinline__ bool place_block(const AttnArgs &p, int *shared, int &b, int &block, int &head, int &rank)
{
    const int task = blockIdx.x / p.S, row_task = task / p.n_kv;
    rank = blockIdx.x % p.S;
    head = task % p.n_kv;
    if (!p.compact) {
        b = row_task % p.n_seq;
        block = p.ntile - 1 - row_task / p.n_seq;
        return true;
    }
    if (threadIdx.x < 32) {
        int x = -1, y = 0;
        if (!find_block(p, row_task, x, y)) x = -1;
        if (threadIdx.x == 0) shared[0] = x, shared[1] = y;
    }
    __syncthreads();
    b = shared[0];
    block = shared[1];
    return b >= 0;
}

template <int DP, int NP>
__global__ void __launch_bounds__(TC_THREADS, 2)
kv8_attn_tc_kernel(const __grid_constant__ AttnArgs p, const int8_t *__restrict__ kc)
{
    using Sh = TcShape<DP, NP>;
    constexpr int DH = DP / 2;                               // dims of a thread
    extern __shared__ uint8_t raw[];
    uint8_t *const tiles = (uint8_t *)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    uint64_t *const bars = (uint64_t *)(tiles + Sh::END);
    uint32_t *const tmem_slot = (uint32_t *)(bars + 2);
    volatile int *const abort = (volatile int *)(tmem_slot + 1);
    float *const xmax = (float *)(tiles + Sh::END + 32);     // [256] a tile's maxima, the two pages of each row
    float *const xsum = xmax + TC_THREADS;
    const int tid = threadIdx.x, warp = tid >> 5, r = tid & 127, h = tid >> 7;
    const uint32_t bar_s = su32(bars), bar_o = su32(bars + 1);
    pdl_wait();
    int b, block_of, head, rank;
    if (!place_block(p, (int *)tmem_slot + 2, b, block_of, head, rank)) return;
    kv8_seq_t seq;
    if (!kv_seq(p.step, b, seq, p.err, tid == 0)) return;
    const int R = seq.n * p.G, r0 = block_of * TC_ROWS;
    if (r0 >= R || R <= p.row_min) return;
    int t0;
    const int np = kv8_tiles(&seq, r0 / p.G, (min(r0 + TC_ROWS, R) - 1) / p.G, p.causal, p.window, rank, p.S, 0, 1, &t0);

    if (tid == 0) {
        bar_init(bar_s, 1);
        bar_init(bar_o, 1);
        *abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(su32(tmem_slot)), "r"(TC_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        // Only now, with its TMEM columns taken, does this CTA let the next kernel start (one thread's signal is the CTA's):
        // a kernel that allocates before it waits for this grid, as the GEMMs do, would otherwise hold columns that this
        // grid waits for. A CTA that returned above needs none.
        lm_signal(p.brief);
    }

    // This thread's row (the last one again where there are fewer) and its keys lo .. hi.
    const int row = min(r0 + r, R - 1), tok = row / p.G;
    const int hi = kv8_hi(&seq, tok, p.causal), lo = kv8_lo(&seq, tok, p.window);
    const long long head_off = (long long)(head * p.G + row % p.G) * p.D;

    // A page's K or V in registers: 16-byte pieces tid and tid + 256. K: a key's pieces side by side, but with 8 of them (D
    // = 128) 8 lanes take the first or last 4 of two keys, which fall into 8 different bank groups when they are stored;
    // V: dim i / 4, keys 16 (i % 4)...
    const int per = p.D / 16, pieces = 4 * p.D;
    int krow[2], kcol[2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
        const int i = tid + TC_THREADS * u;
        krow[u] = per == 8 ? i >> 4 << 1 | (i >> 2 & 1) : i / per;
        kcol[u] = per == 8 ? (i >> 3 & 1) << 2 | (i & 3) : i % per;
    }
    const long long block = (long long)p.D * PAGE;           // bytes of a (page, head)
    auto load_pages = [&](uint4 (&x)[2][2], const int8_t *codes, int a, int z, bool k) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const uint4 *src = (const uint4 *)(codes + ((long long)max(j ? z : a, 0) * p.n_kv + head) * block);
#pragma unroll
            for (int u = 0; u < 2; u++)
                if (tid + TC_THREADS * u < pieces) x[j][u] = __ldg(src + (k ? krow[u] * per + kcol[u] : tid + TC_THREADS * u));
        }
    };
    // page i of this CTA; -1 for none, or one that does not exist
    auto page_at = [&](int i) { return i < np ? kv_page(p.step, b, t0 + i, p.n_pages, p.err, tid == 0) : -1; };
    auto store_k = [&](const uint4 (&x)[2][2]) {
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int u = 0; u < 2; u++)
                if (tid + TC_THREADS * u < pieces)
                    store_codes(tiles + Sh::KV + (kcol[u] >> 2) * Q_TILE, 64 * j + krow[u], 2 * (kcol[u] & 3), x[j][u]);
    };
    auto store_v = [&](const uint4 (&x)[2][2]) {
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int i = tid + TC_THREADS * u;
                if (i < pieces) store_codes(tiles + Sh::KV + j * Sh::V_TILE, i >> 2, 2 * (i & 3), x[j][u]);
            }
    };

    uint4 raw4[2][2] = {};                                   // K of a tile, then its V, then K of the next ...
    int pa = page_at(0), pb = page_at(1), na = page_at(2), nb = page_at(3);   // this tile's pages, and the next's
    load_pages(raw4, kc, pa, pb, true);

    // dims past D are zeros in Q (below); what K and V leave unwritten there only has to be finite
    if (p.D < DP) {
        for (int i = tid; i < (int)(Sh::END - Sh::KV) / 16; i += TC_THREADS)
            *(uint4 *)(tiles + Sh::KV + 16 * i) = make_uint4(0, 0, 0, 0);
    }
    // Q: this thread's half row, scaled by 2^e, as fp16 pieces
    float cs0;
    {
        float x[DH / 16][16], m = 0.0f;
        bool odd = false;
        const long long off = (seq.row0 + tok) * p.ld_q + head_off + DH * h;
#pragma unroll
        for (int c = 0; c < DH / 16; c++) {
#pragma unroll
            for (int e = 0; e < 16; e++) x[c][e] = 0.0f;
            if (DH * h + 16 * c < p.D) load_q16(p, off + 16 * c, x[c]);
        }
#pragma unroll
        for (int c = 0; c < DH / 16; c++) {
#pragma unroll
            for (int e = 0; e < 16; e++) {
                odd |= !(fabsf(x[c][e]) <= 3.402823466e38f);
                m = fmaxf(m, fabsf(x[c][e]));
            }
        }
        xmax[tid] = odd ? __int_as_float(0x7F800000) : m;
        __syncthreads();
        m = fmaxf(xmax[r], xmax[r + 128]);
        odd = !(m <= 3.402823466e38f);
        const int E = (__float_as_int(m) >> 23) & 0xFF;      // the largest magnitude goes to [2^14, 2^15)
        const int e = m == 0.0f ? 0 : max(-126, min(141 - E, 126));
        const float f = odd ? 0.0f : __int_as_float((127 + e) << 23);
        // a row with a NaN or an infinity: zeros here, and a NaN factor
        cs0 = odd ? __int_as_float(0x7FC00000) : p.scale_log2 * __int_as_float((127 - e) << 23);
#pragma unroll
        for (int c = 0; c < DH / 8; c++) {
            const int d = DH * h + 8 * c;
            uint2 a[2], z[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                float y[4];
#pragma unroll
                for (int k = 0; k < 4; k++) y[k] = odd ? 0.0f : x[c / 2][8 * (c & 1) + 4 * i + k];
                f16_pieces4(y, f, a[i], z[i]);
            }
            uint8_t *const q = tiles + Sh::Q + (d >> 6) * Q_TILE + chunk_at(r, (d & 63) >> 3);
            *(uint4 *)q = make_uint4(a[0].x, a[0].y, a[1].x, a[1].y);
            if (NP == 2) *(uint4 *)(q + (DP / 64) * Q_TILE) = make_uint4(z[0].x, z[0].y, z[1].x, z[1].y);
        }
    }
    __syncthreads();                                         // the zeros and the maxima's readers are done
    store_k(raw4);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot, tbase = su32(tiles);
    const uint32_t lane_base = tmem + ((uint32_t)(32 * (warp & 3)) << 16);

    auto issue_s = [&]() {
#pragma unroll
        for (int n = NP - 1; n >= 0; n--)
#pragma unroll
            for (int s = 0; s < DP / 16; s++)
                mma_f16(tmem, sdesc<128>(tbase + Sh::Q + (n * (DP / 64) + (s >> 2)) * Q_TILE + (s & 3) * 32),
                        sdesc<128>(tbase + Sh::KV + (s >> 2) * Q_TILE + (s & 3) * 32), idesc_f16(128),
                        n < NP - 1 || s > 0 ? 1u : 0u);
        mma_commit(bar_s);
    };
    // P of keys 64 j + 32 c + 16 s...: columns 64 j + 32 c + 16 piece + 8 s, the columns that held their scores
    auto issue_o = [&](bool add) {
#pragma unroll
        for (int n = NP - 1; n >= 0; n--)
#pragma unroll
            for (int s = 0; s < 8; s++)
                mma_f16_ts(tmem + 128, tmem + 32 * (s >> 1) + 16 * n + 8 * (s & 1),
                           sdesc<128>(tbase + Sh::KV + (s >> 2) * Sh::V_TILE + (s & 3) * 32), idesc_f16(DP),
                           n < NP - 1 || s > 0 || add ? 1u : 0u);
        mma_commit(bar_o);
    };
    bool ok = true;
    int last_s = -1, last_o = -1;                            // tiles of thread 0's latest commits
    if (tid == 0 && np) {
        issue_s();
        last_s = 0;
    }
    __syncwarp();

    float o[DH], m = -INFINITY, l = 0.0f;                    // m: what O and l stand against; l: this half's share
    float mg = -INFINITY, rest = 0.0f, dm = 0.0f, sv0 = 0.0f;   // the group's references, mg + rest and sv0; dm = mg - 8 - m
#pragma unroll 1
    for (int j = 0; j < DH; j++) o[j] = 0.0f;                // used at a group's end only: kept in local memory
    int left = 0;                                            // tiles that the group may still take
    // The group's P V, complete, joins O; then O and l move to the new m, and a group begins with a tile of maximum t + low.
    auto fold = [&](float t, float low, bool any) {
        const float now = fmaxf(m, t), ref = t < now - FAR_M ? t + ROOM : now, alpha = now == m ? 1.0f : ex2(m - now), f = sv0 * ex2(dm);
#pragma unroll 1
        for (int c = 0; c < DH; c += 32) {
            uint32_t pv[32];
            if (any) tmem_ld32(lane_base + 128 + DH * h + c, pv);
#pragma unroll
            for (int j = 0; j < 32; j++) o[c + j] = alpha * (any ? fmaf(__uint_as_float(pv[j]), f, o[c + j]) : o[c + j]);
        }
        l *= alpha;
        m = now;
        mg = ref;
        rest = ref == t ? low : 0.0f;
        dm = ref == -INFINITY ? 0.0f : ref - now - P_BIAS;   // a row that sees nothing yet has weights of 0
    };
    // log2(s / sv0), also of scales below fp32's normal numbers
    auto log_ratio = [&](float s) {
        const float k = sv0 < 0x1p-60f ? 0x1p64f : 1.0f;
        return __log2f(__fdividef(s * k, sv0 * k));
    };

    // Step it, on tile kb: S is under way. V replaces K when it is done; the maxima are posted and the CTA agrees whether
    // the step opens a group; the weights replace S and P V is issued; when that is done the next step's K replaces V.
    const int tiles_n = (np + 1) / 2;
    bool second = false;                                     // the tile's second page alone
    for (int it = 0, kb = 0; kb < tiles_n; it++) {
        const int mine = h ? pb : pa, key0 = (t0 + 2 * kb + h) * PAGE;
        const long long at_a = (long long)max(pa, 0) * p.n_kv + head, at_b = (long long)max(pb, 0) * p.n_kv + head;
        const float sk = p.k_scale[h ? at_b : at_a];
        const float va = pa < 0 ? 0.0f : p.v_scale[at_a], vb = pb < 0 ? 0.0f : p.v_scale[at_b], sv = h ? vb : va;
        load_pages(raw4, p.v, pa, pb, false);
        const float v_min = fminf(va, vb), v_max = fmaxf(va, vb);
        const bool apart = pa >= 0 && pb >= 0 && v_max > 8.0f * v_min, again = apart && !second;   // the same for the whole CTA
        const bool on = mine >= 0 && (!apart || second == (h != 0));
        const float c = tame(cs0 * (on ? sk : 1.0f));
        float lr = sv == sv0 || !on ? 0.0f : log_ratio(sv);
        const bool whole = __all_sync(0xFFFFFFFFu, on && key0 >= lo && key0 + PAGE - 1 <= hi);
        if (ok) ok = bar_wait(bar_s, (uint32_t)(it & 1), abort, p.err, ERR_WAIT);
        fence_after();
        store_v(raw4);
        // 32 scores of this thread's page, -inf where its row does not see the key
        auto scores = [&](int q, float (&x)[32]) {
            uint32_t s[32];
            tmem_ld32(lane_base + 64 * h + 32 * q, s);
            if (whole) {
#pragma unroll
                for (int j = 0; j < 32; j++) x[j] = __uint_as_float(s[j]);
            } else {
                // bits lo - k0 .. hi - k0, as far as there are such
                const int a = lo - (key0 + 32 * q), z = hi - (key0 + 32 * q);
                const uint32_t from = a <= 0 ? 0xFFFFFFFFu : a > 31 ? 0u : 0xFFFFFFFFu << a;
                const uint32_t upto = z >= 31 ? 0xFFFFFFFFu : z < 0 ? 0u : 0xFFFFFFFFu >> (31 - z);
                const uint32_t sees = on ? from & upto : 0u;
#pragma unroll
                for (int j = 0; j < 32; j++) x[j] = sees >> j & 1u ? __uint_as_float(s[j]) : -INFINITY;
            }
        };
        float top = -INFINITY;
#pragma unroll
        for (int q = 0; q < 2; q++) {
            float x[32];
            scores(q, x);
#pragma unroll
            for (int j = 0; j < 32; j++) top = fmaxf(top, x[j]);
        }
        // The maximum, scaled, is high + low: the product and what its rounding left, which counts where scores pass what
        // 24 bits resolve. A NaN (a NaN query) opens no group.
        const float high = top == -INFINITY ? top : in_range(top * c), low = fabsf(high) < 3e38f ? fmaf(top, c, -high) : 0.0f;
        xmax[tid] = high;
        xsum[tid] = low;
        const bool group = __syncthreads_or(left == 0 || !(fabsf(lr) <= NEAR_V) || high - mg + (low - rest) + lr > GROWTH);
        if (group) {
            const float a = xmax[r], z = xmax[r + 128];
            fold(fmaxf(a, z), a > z ? xsum[r] : a < z ? xsum[r + 128] : fmaxf(xsum[r], xsum[r + 128]), it > 0);
            sv0 = !apart ? v_max : second ? vb : va;
            lr = sv == sv0 || !on ? 0.0f : log_ratio(sv);
            left = NP == 2 ? 4 : 32;
        }
        left--;
        const bool far = fabsf(mg) > FAR_SCORE && mg != -INFINITY;
        const float ref = mg == -INFINITY ? 0.0f : mg, use = P_BIAS + lr - ref;
        float sum = 0.0f;
        auto weights = [&](auto some_far) {
#pragma unroll
            for (int q = 0; q < 2; q++) {
                float x[32];
                uint32_t p1[16], p2[16];
                scores(q, x);
                auto weight = [&](float s) {
                    if (!decltype(some_far)::value || !far) return ex2(fmaf(s, c, use));
                    const float y = fmaf(s, c, -ref) - rest;
                    return ex2((y > GROWTH - lr ? GROWTH - lr : y) + (P_BIAS + lr));    // above only past fp32's range
                };
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    const float a = weight(x[j]), z = weight(x[j + 1]);
                    sum += a + z;
                    const __half2 u = __floats2half2_rn(a, z);
                    p1[j / 2] = *(const uint32_t *)&u;
                    if (NP == 2) {
                        const float2 w = __half22float2(u);
                        const __half2 v = __floats2half2_rn(a - w.x, z - w.y);
                        p2[j / 2] = *(const uint32_t *)&v;
                    }
                }
                if (decltype(some_far)::value) __syncwarp();
                tmem_st16(lane_base + 64 * h + 32 * q, p1);
                if (NP == 2) tmem_st16(lane_base + 64 * h + 32 * q + 16, p2);
            }
        };
        if (__any_sync(0xFFFFFFFFu, far)) weights(std::true_type());
        else weights(std::false_type());
        l = fmaf(sum, ex2(dm - lr), l);
        const bool more = again || kb + 1 < tiles_n;
        if (!again) {
            pa = na, pb = nb;
            na = page_at(2 * kb + 4), nb = page_at(2 * kb + 5);
            kb++;
        }
        second = again;
        if (more) load_pages(raw4, kc, pa, pb, true);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        fence_before();
        __syncthreads();                                     // P and V in place; the maxima and a group's P V read
        fence_after();
        if (tid == 0 && ok) {
            issue_o(!group);
            last_o = it;
        }
        __syncwarp();
        if (ok) ok = bar_wait(bar_o, (uint32_t)(it & 1), abort, p.err, ERR_WAIT);
        fence_after();
        if (more) {
            store_k(raw4);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            fence_before();
            __syncthreads();                                 // the next K in place
            fence_after();
            if (tid == 0 && ok) {
                issue_s();
                last_s = it + 1;
            }
            __syncwarp();
        }
    }
    // The last group's P V joins O on the way out. Where the keys are split, the S CTAs of a cluster took consecutive shares
    // of them: their O (over Q, K and V in shared memory, a row's 16-byte pieces permuted by the row against bank
    // conflicts), m and l meet; each CTA joins every S-th row.
    constexpr int P4 = DP / 4;                               // pieces of a row
    float4 *const po = (float4 *)tiles;
    xsum[tid] = l;
    __syncthreads();
    const float sum = xsum[r] + xsum[r + 128], inv = inverse(sum), last = sv0 * ex2(dm);
    const long long out_off = (seq.row0 + tok) * p.ld_out + head_off + DH * h;
#pragma unroll 1
    for (int c = 0; c < DH; c += 32) {
        uint32_t pv[32] = {};
        if (np > 0) tmem_ld32(lane_base + 128 + DH * h + c, pv);
#pragma unroll
        for (int d = 0; d < 32; d += 4) {
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = fmaf(__uint_as_float(pv[d + e]), last, o[c + d + e]);
            if (p.S > 1) {
                po[r * P4 + ((DH * h + c + d) / 4 ^ (r & (P4 - 1)))] = make_float4(v[0], v[1], v[2], v[3]);
            } else if (ok && r0 + r < R && DH * h + c + d < p.D) {
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] *= inv;
                store_out<4>(p, out_off + c + d, v);
            }
        }
    }
    if (p.S > 1) {
        if (h == 0) {
            xmax[r] = m;
            xmax[r + 128] = sum;
        }
        const uint32_t a_po = su32(po), a_m = su32(xmax);
        cluster_sync();
        const int rows = min(TC_ROWS, R - r0), d4 = p.D / 4;
        auto join = [&](auto most) {
#pragma unroll 4
            for (int i = tid; i < (rows + p.S - 1 - rank) / p.S * d4; i += TC_THREADS) {
                const int k = (int)((unsigned)i * p.d4_inv >> 20), q = rank + k * p.S, d = i - k * d4;
                float v[4];
                cluster_join<decltype(most)::value>(a_m + 4 * q, a_m + 4 * (q + 128), a_po + 16 * (q * P4 + (d ^ (q & (P4 - 1)))),
                                                    p.S, 1.0f, v);
                const int row = r0 + q;
                store_out<4>(p, (seq.row0 + row / p.G) * p.ld_out + (long long)(head * p.G + row % p.G) * p.D + 4 * d, v);
            }
        };
        if (p.S <= 3) join(std::integral_constant<int, 3>());
        else join(std::integral_constant<int, MAX_SPLIT>());
        cluster_sync();                                      // no CTA leaves while another reads its shared memory
    }
    // MMAs that may still run (a wait gave up) must finish before TMEM is freed: thread 0 waits, bounded, for its last
    // commits.
    if (!ok && tid == 0) {
        if (last_s >= 0) bar_wait(bar_s, (uint32_t)(last_s & 1), abort, p.err, ERR_WAIT, false);
        if (last_o >= 0) bar_wait(bar_o, (uint32_t)(last_o & 1), abort, p.err, ERR_WAIT, false);
    }
    fence_before();
    __syncthreads();
    if (warp == 0) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TC_COLS) : "memory");
    }
}

template <int DP, int NP>
bool tc_launch(AttnArgs &p, const int8_t *k, long long R, long long tiles)
{
    using Sh = TcShape<DP, NP>;
    p.ntile = (int)((R + TC_ROWS - 1) / TC_ROWS);
    return attn_grid<kv8_attn_tc_kernel<DP, NP>>(p, dim3(TC_THREADS), Sh::SMEM, TC_ROWS, 2, (tiles + 1) / 2, 1, k);
}

}  // namespace

bool launch_kv8_attn_tc(AttnArgs &p, const int8_t *k, long long R, long long tiles)
{
    if (p.type == GGML_TYPE_F32) return p.D > 64 ? tc_launch<128, 2>(p, k, R, tiles) : tc_launch<64, 2>(p, k, R, tiles);
    return p.D > 64 ? tc_launch<128, 1>(p, k, R, tiles) : tc_launch<64, 1>(p, k, R, tiles);
}

}  // namespace tcg
