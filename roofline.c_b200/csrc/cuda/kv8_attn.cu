// kv8_attn.cu -- attention over the 8-bit key/value cache (tcg_kv8_attention).
//
// For the query rows of one key head (row = token * G + query head of the
// group, G = n_head / n_kv_head) and pages of 64 keys with scales sk, sv:
//   S = Q K^T, P = exp2(c S - m), O = O 2^(m_old - m) + P V, out = O / sum P
// with c = scale log2(e), m the running maximum. Both products run on the
// 8-bit integer tensor path (mma.sync m16n8k32, s32 accumulators), on the
// cache's bytes as they lie there: nothing is converted to a wider type.
//   Q is quantised per row, once, to a whole number of 15 bits (fp16, bf16
//     inputs) or 23 bits (fp32): q = q_scale * (d1 256 + d0), or with d2 65536
//     too, digits of 8 bits in -128 .. 127. The sum over dims is exact.
//   P is taken against the tile's own maximum, so that a tile far below the
//     row's largest score (the rest of a cache beside one key that holds most
//     of the weight) keeps its digits: in [0, 1], it becomes a whole number of
//     16 or 23 bits by one fused multiply-add whose result's mantissa is that
//     number, and byte permutes; P V is exact per tile and folded into fp32
//     with sv 2^(m_tile - m).
// NP = 2 digits leave 2^-16 of a row's largest |q|, NP = 3 2^-24. A weight is
// off by 2^-24 of its tile's largest, and up to 64 of them add up. Two digits
// of P (2^-17) do for 16-bit results only where a tile's weight is spread:
// a row takes them where each of its threads' 16 keys hold 1/16 of its largest
// weight (the other keys then hold 3/16 at least, their 63 roundings 2^-13 of
// that as a rule), three elsewhere, and a warp the third product where one of
// its rows does. Three always: 131071 tokens 52.9
// us against 49.3 with scores of spread 2.7, 64 x 16 rows 136 against 133.
//
// Why no shuffles: the mma's k order is free as long as A and B agree. A
// thread (row g = lane / 4, t = lane % 4) takes 16 consecutive bytes of a K
// row or of a V row (V is stored dim-major) as one 128-bit shared-memory word
// for four k-quads; key 16 t + 2 j + c is column 2 t + c of score tile j, so
// the scores a thread holds are exactly the P bytes its own A fragments need.
//
// A tile is one page's K block (64 keys x D, a TMA box per 64 dims, zeros past
// D) and V block (D x 64, one bulk copy); K and V tiles alternate through a
// ring of slots, each with an mbarrier. The last warp to release a slot issues
// the copy that refills it, so there is no producer warp.
//
// Rows of a warp: 16 (RW = 2), or 8 (RW = 1) with the two upper digits of Q,
// and of P, as rows g and g + 8 of one A operand (a second one holds the third
// digit). A decode step has few rows (G, often 4 or 8): 8 of them then cost
// half the MMAs, accumulators and registers (64 sequences up to 8192 tokens,
// bf16: 137 -> 109 us; one token over 131071: 88 -> 61 us).
//
// Work split: WM warps take their rows of the same tiles, WN groups of warps
// take alternate tiles, and a cluster of S CTAs takes S consecutive shares of
// the keys; partial results (m, l, O) meet in shared memory, then over
// distributed shared memory, in a fixed order. No workspace, one launch. 12
// warps an SM with two slots each beat 8 with three (131071 tokens at S = 8:
// 53.3 against 61.1 us): the warps' own latency, not the copies in flight,
// was the limit.
//
// Bound by memory on large decode batches: 64 sequences up to 8192 tokens (32
// query heads, 8 key heads, D = 128) 105 us, 6.1 TB/s. One token over 131071:
// 48 us, 5.5 TB/s: clusters of 10 use 80 of 148 SMs. One token over a few
// hundred: 6.3 us (bf16) to 6.8 us (fp32), an empty kernel launched the same
// way 2.6 us; dependent loads (lengths, page,
// scale and tile) and the launch.
#include "kv8_attn.cuh"
#include "tc05.cuh"

#include <math.h>

#include <atomic>
#include <type_traits>

namespace tcg {
namespace {

__device__ __forceinline__ void mma_s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_u8s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 lds128(uint32_t a)
{
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// 4 consecutive values of a query row.
__device__ __forceinline__ void load_q4(const AttnArgs &p, long long off, float (&x)[4])
{
    if (p.type == GGML_TYPE_F32) {
        const float *s = (const float *)p.q + off;
        if (p.q_vec) load_pack<float, 4>(s, x);
        else
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = s[e];
        return;
    }
    const unsigned short *s = (const unsigned short *)p.q + off;
    ushort4 v;
    if (p.q_vec) v = *(const ushort4 *)s;
    else v = make_ushort4(s[0], s[1], s[2], s[3]);
    const unsigned short h[4] = { v.x, v.y, v.z, v.w };
#pragma unroll
    for (int e = 0; e < 4; e++)
        x[e] = p.type == GGML_TYPE_BF16 ? __uint_as_float((uint32_t)h[e] << 16) : __half2float(__ushort_as_half(h[e]));
}

// O is kept times this, about the root of what a weight's digits count to: the factor of a tile's P V (its V scale over
// that count) then keeps its bits down to V of 1e-33, and the sums have room up to 1e35. At 1 it lost them below 1e-29.
constexpr float O_UNIT = 2048.0f;

// What a weight of 1 is as a whole number of 23 and 16 bits. Below 2^23 by more than ex2's error and the product's
// rounding up to FAR_SCORE, 2^-12 of the weight at most, can put it above 1: a weight past the last number would be 0.
constexpr float P3 = 8386000.0f, P2 = 65516.0f;

template <int KS, int NP, int RW, int WM, int WN, int NSLOT>
struct Shape {
    static constexpr int DP = KS * 32;                       // dims, padded
    static constexpr int SLOT = PAGE * DP;                   // bytes of a K or V tile
    static constexpr int RING = WN * NSLOT * SLOT;
    static constexpr int ROWS = 8 * RW * WM;
    static constexpr int PITCH = DP + 8;                     // floats of a partial O row
    static constexpr int EXCH = (WN * ROWS * (PITCH + 2) + 2 * ROWS) * 4;    // partial O, m, l; the CTA's m, l
    static constexpr int BODY = RING > EXCH ? RING : EXCH;
    static constexpr int Q_PITCH = DP / 4 + 4;               // words of a row of Q digits: 8 rows in 8 bank groups
    static constexpr int QROWS = WN > 1 ? ROWS : 0;          // digits, factors, barriers
    static constexpr int QD = BODY, QS = QD + NP * QROWS * Q_PITCH * 4, BARS = QS + QROWS * 4;
    static_assert(BODY % 16 == 0 && BARS % 16 == 0, "alignment");
    static constexpr size_t SMEM = 128 + BARS + WN * NSLOT * 12 + 16;
};

template <int KS, int NP, int RW, int WM, int WN, int NSLOT, int MINB>
__global__ void __launch_bounds__(32 * WM * WN, MINB)
kv8_attn_kernel(const __grid_constant__ AttnArgs p, const __grid_constant__ CUtensorMap kmap)
{
    using Sh = Shape<KS, NP, RW, WM, WN, NSLOT>;
    constexpr int NT = KS * 4;                               // 8-dim output tiles
    extern __shared__ uint8_t raw[];
    uint8_t *const base = (uint8_t *)(((uintptr_t)raw + 127) & ~(uintptr_t)127);
    const uint32_t ring = su32(base), bars = ring + Sh::BARS;
    int *const count = (int *)(base + Sh::BARS + WN * NSLOT * 8);
    volatile int *const abort = (volatile int *)(count + WN * NSLOT);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int wm = warp % WM, wn = warp / WM;

    if (threadIdx.x == 0) {
        for (int i = 0; i < WN * NSLOT; i++) {
            bar_init(bars + 8 * i, 1);
            count[i] = 0;
        }
        *abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    lm_begin(p.brief);
    const int rank = blockIdx.x % p.S, head = blockIdx.x / p.S % p.n_kv, b = blockIdx.x / p.S / p.n_kv;

    // Where the tiles start at key 0 and are this CTA's alone, the first pages are asked for along with the lengths; an
    // entry behind the sequence's end is not used.
    const bool from0 = p.S == 1 && !p.window;
    const int ahead = wn + lane * WN, guess = from0 && ahead < p.step.table_ld ? p.step.table[(size_t)b * p.step.table_ld + ahead] : -1;
    kv8_seq_t seq;
    const bool report = threadIdx.x == 0;
    if (!kv_seq(p.step, b, seq, p.err, report)) return;      // the same for the whole cluster
    const int R = seq.n * p.G;                               // one block holds them: the host picks a shape by the longest
    if (R == 0 || R > Sh::ROWS) return;
    auto tok_of = [&](int r) { return (int)((unsigned)r * p.g_inv >> 20); };   // r / G, for r < 64
    auto hi_of = [&](int tok) { return kv8_hi(&seq, tok, p.causal); };
    auto lo_of = [&](int tok) { return kv8_lo(&seq, tok, p.window); };
    int t0;                                                  // this warp group's tiles: t0, t0 + WN, ...
    const int mine = kv8_tiles(&seq, 0, tok_of(R - 1), p.causal, p.window, rank, p.S, wn, WN, &t0);

    // This thread's rows.
    constexpr int RPW = 8 * RW;                              // rows of a warp
    int hi[RW], lo[RW];
    long long row_off[RW];
#pragma unroll
    for (int i = 0; i < RW; i++) {
        const int r = min(RPW * wm + g + 8 * i, R - 1), tok = tok_of(r);
        hi[i] = hi_of(tok);
        lo[i] = lo_of(tok);
        row_off[i] = (long long)(head * p.G + r - tok * p.G) * p.D;
    }
    const int row_a = tok_of(min(RPW * wm, R - 1)), row_z = tok_of(min(RPW * wm + RPW - 1, R - 1));
    const int all_hi = hi_of(row_a), all_lo = lo_of(row_z);  // keys that every row of the warp sees
    const int any_hi = hi_of(row_z), any_lo = lo_of(row_a);  // keys that some row of the warp sees

    // Pages and scales of 32 tiles at a time, one per lane; the next 32 pages too.
    auto page_at = [&](int i) {
        return i < mine ? kv_page(p.step, b, t0 + i * WN, p.n_pages, p.err, true) : 0;
    };
    int page = guess, page_next = page_at(32 + lane);
    if (!from0 || (lane < mine && !kv8_page_ok(guess, p.n_pages))) page = page_at(lane);   // with its error, if it is one
    if (lane >= mine) page = 0;
    float sk = 0.0f, sv = 0.0f;
    auto scales = [&]() {
        const long long at = (long long)max(page, 0) * p.n_kv + head;
        sk = p.k_scale[at];
        sv = p.v_scale[at];
    };

    const uint32_t my_ring = ring + wn * NSLOT * Sh::SLOT, my_bars = bars + wn * NSLOT * 8;
    int *const my_count = count + wn * NSLOT;
    // Item n = K (even) or V (odd) of tile n / 2, into slot n % NSLOT. A page that does not exist is masked; its copy
    // takes page 0 instead.
    auto issue = [&](int n, int slot, int pg) {
        const uint32_t dst = my_ring + slot * Sh::SLOT, bar = my_bars + 8 * slot;
        const long long at = (long long)max(pg, 0) * p.n_kv + head;
        if (n & 1) {
            const uint32_t bytes = (uint32_t)p.D * PAGE;
            bar_expect_tx(bar, bytes);
            bulk_load(dst, p.v + at * p.D * PAGE, bytes, bar);
        } else {
            bar_expect_tx(bar, Sh::SLOT);
#pragma unroll
            for (int c = 0; c < KS / 2; c++) tma_load(dst + c * 4096, &kmap, bar, 64 * c, (int)(at * PAGE));
        }
    };
    auto page_of = [&](int i, int now) {                     // whole warp
        return __shfl_sync(0xFFFFFFFFu, (i >> 5) == (now >> 5) ? page : page_next, i & 31);
    };
    if (wm == 0) {
#pragma unroll
        for (int n = 0; n < NSLOT; n++) {
            const int pg = page_of(n >> 1, 0);
            if (lane == 0 && n < 2 * mine) issue(n, n, pg);
        }
    }
    scales();

    // A fragments, in the k order of the tiles: k-step 2 c + s of chunk c takes bytes 64 c + 16 t + 8 s + 0..7. RW = 2:
    // qd[n] is digit n's. RW = 1: the first fragment holds the two upper digits, as rows g and g + 8; with three digits a
    // second one holds the lowest as row g + 8.
    constexpr int NA = RW == 2 ? NP : NP - 1;                // A fragments, mma's of Q K^T
    constexpr int NAP = RW == 2 ? 3 : 2;                     // the same of P V, which takes up to three digits
    uint32_t qd[NA][KS][4] = {};
    float qs[RW];
    constexpr float Q = NP == 3 ? 8300000.0f : 32512.0f;     // the digits' largest sums
    if constexpr (WN == 1) {
        // each thread the digits of its own fragments
#pragma unroll
        for (int i = 0; i < RW; i++) {
            float x[KS / 2][16], m = 0.0f;
            bool odd = false;                                    // a NaN or an infinity
            const int r = min(RPW * wm + g + 8 * i, R - 1);
            const long long off = (seq.row0 + tok_of(r)) * p.ld_q + row_off[i];
#pragma unroll
            for (int c = 0; c < KS / 2; c++) {
#pragma unroll
                for (int e = 0; e < 16; e++) x[c][e] = 0.0f;
                if (64 * c + 16 * t < p.D) load_q16(p, off + 64 * c + 16 * t, x[c]);
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    odd |= !(fabsf(x[c][e]) <= 3.402823466e38f);
                    m = fmaxf(m, fabsf(x[c][e]));
                }
            }
            m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
            m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
            odd = odd | __shfl_xor_sync(0xFFFFFFFFu, (int)odd, 1);
            odd = odd | __shfl_xor_sync(0xFFFFFFFFu, (int)odd, 2);
            const float lift = m < 1e-20f ? 0x1p80f : 1.0f;      // keeps Q / m finite
            const double back = m < 1e-20f ? 0x1p-80 : 1.0;
            m = fmaxf(m * lift, 1e-21f);
            const float up = Q / m;
            qs[i] = odd ? __int_as_float(0x7FC00000) : (float)fmin((double)m * back * (double)p.scale_log2 * (1.0 / Q), 3e38);
#pragma unroll
            for (int c = 0; c < KS / 2; c++)
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    uint32_t d[NP] = {};
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        int v = __float2int_rn(x[c][4 * w + e] * lift * up);
#pragma unroll
                        for (int n = 0; n < NP; n++) {
                            const int dig = (int)(int8_t)v;
                            d[n] |= (uint32_t)(dig & 0xFF) << (8 * e);
                            v = (v - dig) >> 8;
                        }
                    }
                    if (RW == 2) {
#pragma unroll
                        for (int n = 0; n < NP; n++) qd[n % NA][2 * c + (w >> 1)][2 * (w & 1) + i] = d[n];
                    } else {
                        qd[0][2 * c + (w >> 1)][2 * (w & 1)] = d[NP - 1];
                        qd[0][2 * c + (w >> 1)][2 * (w & 1) + 1] = d[NP - 2];
                        if (NP == 3) qd[NA - 1][2 * c + (w >> 1)][2 * (w & 1) + 1] = d[0];
                    }
                }
        }
    } else {
        // The WN groups need the same digits: a warp a row, 4 dims a lane, through shared memory (one token over 513, fp32:
        // 8.5 -> 7.1 us). With one group the shuffles cost more than they save (64 x 16 rows, bf16: 148 against 123 us).
        uint32_t *const sq = (uint32_t *)(base + Sh::QD);        // [NP][ROWS][Q_PITCH], lowest digit first
        float *const sqs = (float *)(base + Sh::QS);
        constexpr int EACH = (Sh::ROWS + WM * WN - 1) / (WM * WN), AT_ONCE = EACH < 8 ? EACH : 8;   // rows whose loads go together
        static_assert(EACH <= 32, "a lane keeps what belongs to one of the warp's rows");
        const int my_row = min(warp + lane * WM * WN, R - 1);    // of the warp's lane-th row: where it lies, its largest value
        const int my_tok = tok_of(my_row);
        const long long my_off = (seq.row0 + my_tok) * p.ld_q + (long long)(head * p.G + my_row - my_tok * p.G) * p.D;
        float my_max = 0.0f;
#pragma unroll
        for (int k0 = 0; k0 < EACH; k0 += AT_ONCE) {
            float x[AT_ONCE][4] = {};
#pragma unroll
            for (int k = 0; k < AT_ONCE; k++) {
                const long long off = __shfl_sync(0xFFFFFFFFu, my_off, k0 + k);
                if (4 * lane < p.D) load_q4(p, off + 4 * lane, x[k]);
            }
#pragma unroll
            for (int k = 0; k < AT_ONCE; k++) {
                const int r = warp + (k0 + k) * WM * WN;
                float m = fmaxf(fmaxf(fabsf(x[k][0]), fabsf(x[k][1])), fmaxf(fabsf(x[k][2]), fabsf(x[k][3])));
                // NaN where the row has a NaN or an infinity: fmaxf drops a NaN, the sum of x * 0 does not
                m += (x[k][0] * 0.0f + x[k][1] * 0.0f) + (x[k][2] * 0.0f + x[k][3] * 0.0f);
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    const float y = __shfl_xor_sync(0xFFFFFFFFu, m, o);
                    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(m), "f"(y));
                }
                my_max = lane == k0 + k ? m : my_max;
                const float lift = m < 1e-20f ? 0x1p80f : 1.0f, up = Q / fmaxf(m * lift, 1e-21f);   // lift keeps Q / m finite
                uint32_t d[NP] = {};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    int v = __float2int_rn(x[k][e] * lift * up);
#pragma unroll
                    for (int n = 0; n < NP; n++) {
                        const int dig = (int)(int8_t)v;
                        d[n] |= (uint32_t)(dig & 0xFF) << (8 * e);
                        v = (v - dig) >> 8;
                    }
                }
                if (r < Sh::ROWS && 4 * lane < Sh::DP)
#pragma unroll
                    for (int n = 0; n < NP; n++) sq[(n * Sh::ROWS + r) * Sh::Q_PITCH + lane] = d[n];
            }
        }
        if (lane < EACH && warp + lane * WM * WN < Sh::ROWS) {
            // the factor of the row: NaN stays NaN
            const double m = my_max < 1e-20f ? fmax((double)my_max * 0x1p80, 1e-21) * 0x1p-80 : (double)my_max;
            const double s = m * (double)p.scale_log2 * (1.0 / Q);
            sqs[warp + lane * WM * WN] = (float)(s > 3e38 ? 3e38 : s);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < RW; i++) {
            const int r = RPW * wm + g + 8 * i;
            qs[i] = sqs[r];
#pragma unroll
            for (int n = 0; n < NP; n++)
#pragma unroll
                for (int c = 0; c < KS / 2; c++) {
                    const uint4 v = *(const uint4 *)(sq + (n * Sh::ROWS + r) * Sh::Q_PITCH + 16 * c + 4 * t);
                    const uint32_t w[4] = { v.x, v.y, v.z, v.w };
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        if (RW == 2) qd[n % NA][2 * c + (k >> 1)][2 * (k & 1) + i] = w[k];
                        else if (n == NP - 1) qd[0][2 * c + (k >> 1)][2 * (k & 1)] = w[k];
                        else if (n == NP - 2) qd[0][2 * c + (k >> 1)][2 * (k & 1) + 1] = w[k];
                        else qd[NA - 1][2 * c + (k >> 1)][2 * (k & 1) + 1] = w[k];
                    }
                }
        }
    }

    float o[NT][2 * RW], m[RW], l[RW];
#pragma unroll
    for (int i = 0; i < RW; i++) {
        m[i] = -INFINITY;
        l[i] = 0.0f;
    }
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 2 * RW; e++) o[n][e] = 0.0f;

    int slot = 0, parity = 0;
    bool ok = true;
    // Whole warp: this warp is done with item n in `slot`; whoever is last refills it.
    auto release = [&](int n) {
        const int next = n + NSLOT, pg = page_of(next >> 1, n >> 1);
        __syncwarp();
        if (lane == 0) {
            bool last = true;
            if (WM > 1) {
                __threadfence_block();
                last = atomicAdd(my_count + slot, 1) == WM - 1;
                if (last) {
                    my_count[slot] = 0;
                    __threadfence_block();
                }
            }
            if (last && next < 2 * mine) {
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                issue(next, slot, pg);
            }
        }
        if (++slot == NSLOT) {
            slot = 0;
            parity ^= 1;
        }
    };
    auto landed = [&]() {
        return __all_sync(0xFFFFFFFFu, bar_wait(my_bars + 8 * slot, parity, abort, p.err, ERR_WAIT));
    };

    for (int i = 0; i < mine; i++) {
        if (i && (i & 31) == 0) {
            page = page_next;
            page_next = page_at(i + 32 + lane);
            scales();
        }
        const int key0 = (t0 + i * WN) * PAGE;
        const bool real = __shfl_sync(0xFFFFFFFFu, page, i & 31) >= 0 && key0 <= any_hi && key0 + PAGE > any_lo;
        const float tk = __shfl_sync(0xFFFFFFFFu, sk, i & 31), tv = __shfl_sync(0xFFFFFFFFu, sv, i & 31);

        ok = landed();
        if (!ok) break;
        float f[8][2 * RW];
        if (real) {
            const uint32_t kt = my_ring + slot * Sh::SLOT + (16 * (g >> 1) + (g & 1)) * 64 + 16 * t;
            constexpr int B = 4;                             // score tiles side by side: independent mma chains
#pragma unroll
            for (int j0 = 0; j0 < 8; j0 += B) {
                uint4 w[KS / 2][B];
                int a[B][4] = {}, top[B][4] = {};
#pragma unroll
                for (int c = 0; c < KS / 2; c++)
#pragma unroll
                    for (int j = 0; j < B; j++) w[c][j] = lds128(kt + c * 4096 + (j0 + j) * 128);
                auto dims = [&](int (&d)[B][4], const uint32_t (&q)[KS][4]) {
#pragma unroll
                    for (int c = 0; c < KS / 2; c++) {
#pragma unroll
                        for (int j = 0; j < B; j++) mma_s8(d[j], q[2 * c], w[c][j].x, w[c][j].y);
#pragma unroll
                        for (int j = 0; j < B; j++) mma_s8(d[j], q[2 * c + 1], w[c][j].z, w[c][j].w);
                    }
                };
                if constexpr (RW == 2) {
                    dims(a, qd[1]);
                    if (NP == 3) dims(top, qd[NA - 1]);
#pragma unroll
                    for (int j = 0; j < B; j++)
#pragma unroll
                        for (int e = 0; e < 4; e++) a[j][e] <<= 8;   // |a| < 2^21 (128 dims): below 2^30 with the next digit
                    dims(a, qd[0]);
#pragma unroll
                    for (int j = 0; j < B; j++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            f[j0 + j][e] = NP == 3 ? fmaf((float)top[j][e], 65536.0f, (float)a[j][e]) : (float)a[j][e];
                } else {
                    dims(a, qd[0]);
                    if (NP == 3) {
#pragma unroll
                        for (int j = 0; j < B; j++) a[j][2] <<= 8, a[j][3] <<= 8;
                        dims(a, qd[NA - 1]);                 // its rows 0..7 are zero
                    }
#pragma unroll
                    for (int j = 0; j < B; j++)
#pragma unroll
                        for (int e = 0; e < 2; e++)
                            f[j0 + j][e] = NP == 3 ? fmaf((float)a[j][e], 65536.0f, (float)a[j][2 + e])
                                                   : (float)(a[j][e] * 256 + a[j][2 + e]);
                }
            }
        }
        release(2 * i);

        uint32_t pd[NAP][2][4] = {};
        float fold[RW];                                      // factor of the tile's P V, into O
        bool fine = true;                                    // three digits of P
        if (real) {
            if (key0 < all_lo || key0 + PAGE - 1 > all_hi) {
#pragma unroll
                for (int j = 0; j < 8; j++)
#pragma unroll
                    for (int e = 0; e < 2 * RW; e++) {
                        const int key = key0 + 16 * t + 2 * j + (e & 1);
                        if (key > hi[e >> 1] || key < lo[e >> 1]) f[j][e] = -INFINITY;
                    }
            }
            bool grew = false;
            uint32_t spread[RW];                             // lanes whose 16 keys hold 1/16 of their row's largest weight
            float up[RW];                                    // of O, where the row's maximum grew
#pragma unroll
            for (int r = 0; r < RW; r++) {
                float top = -INFINITY;
#pragma unroll
                for (int j = 0; j < 8; j++) top = fmaxf(top, fmaxf(f[j][2 * r], f[j][2 * r + 1]));
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                float cs = tame(qs[r] * tk);
                const bool none = top == -INFINITY, far = !none && fabsf(top * cs) > FAR_SCORE;
                const float mt = none ? top : in_range(top * cs);
                float ref = none ? 0.0f : mt;
                const float mn = fmaxf(m[r], mt), use = mn == -INFINITY ? 0.0f : mn;
                const float beta = ex2(mt - use);
                up[r] = ex2(m[r] - use);
                grew |= mn != m[r];
                m[r] = mn;
                if (far) {
#pragma unroll
                    for (int j = 0; j < 8; j++)
#pragma unroll
                        for (int c = 0; c < 2; c++) f[j][2 * r + c] = (f[j][2 * r + c] - top) * cs;
                    cs = 1.0f, ref = 0.0f;
                }
                float sum = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; j++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        float &v = f[j][2 * r + c];
                        v = ex2(fmaf(v, cs, -ref));
                        sum += v;
                    }
                l[r] = fmaf(l[r], up[r], sum * beta);
                fold[r] = tv * beta;
                spread[r] = NP == 3 ? 0 : __ballot_sync(0xFFFFFFFFu, !(sum < 1.0f / 16.0f));
            }
            fine = (spread[0] & spread[RW - 1]) != 0xFFFFFFFFu;
            if (__any_sync(0xFFFFFFFFu, grew)) {
#pragma unroll
                for (int r = 0; r < RW; r++)
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        o[n][2 * r] *= up[r];
                        o[n][2 * r + 1] *= up[r];
                    }
            }
            // bytes of the four weights of keys 16 t + 4 w + 0..3
            auto digits = [&](auto three) {
                constexpr bool THREE = decltype(three)::value;
#pragma unroll
                for (int r = 0; r < RW; r++) {
                    // each row its own digits, whatever its neighbours need: two of them are three with a zero
                    const bool mine = THREE && (NP == 3 || (spread[r] >> (lane & 28) & 15u) != 15u);
                    const float one = mine ? P3 : P2 / 65536.0f, base_of = mine ? 8388608.0f : 128.0f;
                    fold[r] *= mine ? O_UNIT / P3 : O_UNIT / P2;
#pragma unroll
                    for (int w = 0; w < 4; w++) {
                        uint32_t y[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const float v = f[2 * w + (e >> 1)][2 * r + (e & 1)];
                            y[e] = __float_as_uint(fmaf(v, one, base_of));
                        }
                        const uint32_t u = __byte_perm(y[0], y[1], 0x5140), v = __byte_perm(y[2], y[3], 0x5140);
                        const uint32_t d0 = __byte_perm(u, v, 0x5410), d1 = __byte_perm(u, v, 0x7632);
                        const uint32_t d2 = __byte_perm(__byte_perm(y[0], y[1], 0x0062), __byte_perm(y[2], y[3], 0x0062), 0x5410);
                        const int at = 2 * (w & 1);
                        if constexpr (RW == 2) {
                            pd[0][w >> 1][at + r] = d0;
                            pd[1][w >> 1][at + r] = d1;
                            if (THREE) pd[NAP - 1][w >> 1][at + r] = d2;
                        } else {
                            pd[0][w >> 1][at] = THREE ? d2 : d1;
                            pd[0][w >> 1][at + 1] = THREE ? d1 : d0;
                            if (THREE) pd[1][w >> 1][at + 1] = d0;
                        }
                    }
                }
            };
            if (NP == 3 || fine) digits(std::true_type());
            else digits(std::false_type());
        }

        ok = landed();
        if (!ok) break;
        if (real) {
            const uint32_t vt = my_ring + slot * Sh::SLOT + g * 64 + 16 * t;
            constexpr int B = 4;                             // output tiles side by side
            auto product = [&](auto three) {
                constexpr bool THREE = decltype(three)::value;
#pragma unroll
                for (int n0 = 0; n0 < NT; n0 += B) {
                    uint4 w[B];
                    int a[B][4] = {}, top[B][4] = {};
#pragma unroll
                    for (int n = 0; n < B; n++) w[n] = lds128(vt + (n0 + n) * 512);
                    auto keys = [&](int (&d)[B][4], const uint32_t (&q)[2][4]) {
#pragma unroll
                        for (int n = 0; n < B; n++) mma_u8s8(d[n], q[0], w[n].x, w[n].y);
#pragma unroll
                        for (int n = 0; n < B; n++) mma_u8s8(d[n], q[1], w[n].z, w[n].w);
                    };
                    if constexpr (RW == 2) {
                        keys(a, pd[1]);
                        if (THREE) keys(top, pd[NAP - 1]);
#pragma unroll
                        for (int n = 0; n < B; n++)
#pragma unroll
                            for (int e = 0; e < 4; e++) a[n][e] <<= 8;   // |a| <= 255 * 128 * 64 < 2^21
                        keys(a, pd[0]);
#pragma unroll
                        for (int n = 0; n < B; n++)
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                o[n0 + n][e] = fmaf(THREE ? fmaf((float)top[n][e], 65536.0f, (float)a[n][e]) : (float)a[n][e],
                                                    fold[e >> 1], o[n0 + n][e]);
                    } else {
                        keys(a, pd[0]);
                        if (THREE) {
#pragma unroll
                            for (int n = 0; n < B; n++) a[n][2] <<= 8, a[n][3] <<= 8;
                            keys(a, pd[1]);                  // its rows 0..7 are zero
                        }
#pragma unroll
                        for (int n = 0; n < B; n++)
#pragma unroll
                            for (int e = 0; e < 2; e++)
                                o[n0 + n][e] = fmaf(THREE ? fmaf((float)a[n][e], 65536.0f, (float)a[n][2 + e])
                                                          : (float)(a[n][e] * 256 + a[n][2 + e]), fold[0], o[n0 + n][e]);
                    }
                }
            };
            if (NP == 3 || fine) product(std::true_type());
            else product(std::false_type());
        }
        release(2 * i + 1);
    }

#pragma unroll
    for (int r = 0; r < RW; r++) {
        l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], 1);
        l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], 2);
    }

    if (!ok) {
        // A copy did not land in time: the error word is set. Nothing is reused; each group waits, bounded, for the
        // copies it has in flight before the CTA may end (or its ring be overwritten).
        for (int s = 0; s < NSLOT; s++) bar_wait(my_bars + 8 * s, parity ^ (s < slot), abort, p.err, ERR_WAIT, false);
    }
    if (WN == 1 && p.S == 1) {
#pragma unroll
        for (int r = 0; r < RW; r++) {
            const int row = RPW * wm + g + 8 * r;
            if (row >= R) continue;
            const float inv = inverse(l[r]) * (1.0f / O_UNIT);
            const long long off = (seq.row0 + tok_of(row)) * p.ld_out + row_off[r];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                if (8 * n >= p.D) break;
                const float v[2] = { o[n][2 * r] * inv, o[n][2 * r + 1] * inv };
                store_out<2>(p, off + 8 * n + 2 * t, v);
            }
        }
        return;
    }

    // Partial results meet: the WN groups of this CTA, then the S CTAs of the cluster.
    __syncthreads();                                         // every tile is consumed: the ring is free
    float *const po = (float *)base;                         // [WN][ROWS][PITCH]
    float *const pm = po + WN * Sh::ROWS * Sh::PITCH;        // [WN][ROWS]
    float *const pl = pm + WN * Sh::ROWS;
    float *const qm = pl + WN * Sh::ROWS;                    // [ROWS] the CTA's
    float *const ql = qm + Sh::ROWS;
    const int rows = R, d4 = p.D / 4;
#pragma unroll
    for (int r = 0; r < RW; r++) {
        const int at = wn * Sh::ROWS + RPW * wm + g + 8 * r;
#pragma unroll
        for (int n = 0; n < NT; n++)
            *(float2 *)(po + at * Sh::PITCH + 8 * n + 2 * t) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
        if (t == 0) {
            pm[at] = m[r];
            pl[at] = l[r];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows * d4; i += blockDim.x) {
        const int r = (int)((unsigned)i * p.d4_inv >> 20), d = 4 * (i - r * d4);
        float top = -INFINITY, sum = 0.0f, v[4] = {};
#pragma unroll
        for (int w = 0; w < WN; w++) top = fmaxf(top, pm[w * Sh::ROWS + r]);
        const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int w = 0; w < WN; w++) {
            const float a = ex2(pm[w * Sh::ROWS + r] - ref);
            const float4 x = *(const float4 *)(po + (w * Sh::ROWS + r) * Sh::PITCH + d);
            sum = fmaf(a, pl[w * Sh::ROWS + r], sum);
            v[0] = fmaf(a, x.x, v[0]), v[1] = fmaf(a, x.y, v[1]), v[2] = fmaf(a, x.z, v[2]), v[3] = fmaf(a, x.w, v[3]);
        }
        if (p.S > 1) {                                       // to group 0's place: this thread alone reads it
            *(float4 *)(po + r * Sh::PITCH + d) = make_float4(v[0], v[1], v[2], v[3]);
            if (d == 0) qm[r] = top, ql[r] = sum;
            continue;
        }
        const float inv = inverse(sum) * (1.0f / O_UNIT);
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] *= inv;
        store_out<4>(p, (seq.row0 + tok_of(r)) * p.ld_out + (long long)(head * p.G + r - tok_of(r) * p.G) * p.D + d, v);
    }
    if (p.S == 1) return;
    const uint32_t a_po = su32(po), a_qm = su32(qm), a_ql = su32(ql);
    cluster_sync();
    for (int i = threadIdx.x + rank * blockDim.x; i < rows * d4; i += blockDim.x * p.S) {
        const int r = (int)((unsigned)i * p.d4_inv >> 20), d = 4 * (i - r * d4);
        float v[4];
        cluster_join<MAX_SPLIT>(a_qm + 4 * r, a_ql + 4 * r, a_po + 4 * (r * Sh::PITCH + d), p.S, 1.0f / O_UNIT, v);
        store_out<4>(p, (seq.row0 + tok_of(r)) * p.ld_out + (long long)(head * p.G + r - tok_of(r) * p.G) * p.D + d, v);
    }
    cluster_sync();                                          // no CTA leaves while another reads its shared memory
}


typedef CUresult (*EncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                             const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                             CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn attn_encode_fn()
{
    static std::atomic<EncodeFn> known{nullptr};             // threads that come first together find the same
    EncodeFn fn = known.load(std::memory_order_acquire);
    if (!fn) {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            known.store(fn = (EncodeFn)p, std::memory_order_release);
        else
            cudaGetLastError();
    }
    return fn;
}

template <int KS, int NP, int RW, int WM, int WN, int NSLOT, int MINB>
bool attn_launch(AttnArgs &p, const CUtensorMap &map, long long tiles)
{
    using Sh = Shape<KS, NP, RW, WM, WN, NSLOT>;
    p.ntile = 1;
    return attn_grid<kv8_attn_kernel<KS, NP, RW, WM, WN, NSLOT, MINB>>(p, dim3(32 * WM * WN), Sh::SMEM, Sh::ROWS, MINB, tiles, WN, map);
}

}  // namespace
}  // namespace tcg

using namespace tcg;

extern "C" bool tcg_kv8_attention(void *out, const void *q, const tcg_kv8_t *c, const tcg_kv8_step_t *s, int n_head,
                                  int64_t ld_out, int64_t ld_q, float scale, bool causal, int window, ggml_type_t t)
{
    const char *who = "tcg_kv8_attention";
    if (!kv8_check(who, c, s, t)) return false;
    if (n_head < 1 || n_head % c->n_kv_head || n_head / c->n_kv_head > 4096)
        return fail("%s: %d query heads over %d key heads", who, n_head, c->n_kv_head);
    if (!(scale > 0.0f) || scale > 1e30f) return fail("%s: scale %g is not positive", who, (double)scale);
    if (window < 0 || (window && !causal)) return fail("%s: window %d%s", who, window, causal ? "" : " without causal");
    const size_t size = lm_type_size(t);
    if (s->n_tok && (!out || !q)) return fail("%s: no queries or no output", who);
    if (((uintptr_t)out | (uintptr_t)q) % size) return fail("%s: misaligned queries or output", who);
    const int64_t wide = (int64_t)n_head * c->head_dim;
    if ((ld_q < wide || ld_out < wide) && s->n_tok > 1)
        return fail("%s: rows of %lld values do not fit strides of %lld and %lld", who, (long long)wide, (long long)ld_q,
                    (long long)ld_out);

    const int longest = s->max_new < s->n_tok ? s->max_new : s->n_tok, G = n_head / c->n_kv_head;
    const long long R = (long long)(longest > 0 ? longest : 1) * G;
    if (R > 0x3fffffffll) return fail("%s: %d rows of %d heads are too many for one call", who, longest, n_head);
    if (!lm_ready(who)) return false;
    if (s->n_seq == 0 || s->n_tok == 0) return true;
    AttnArgs p = {};
    p.q = q, p.out = out, p.ld_q = ld_q, p.ld_out = ld_out, p.type = (int)t;
    p.q_vec = (uintptr_t)q % 16 == 0 && ld_q * (int64_t)size % 16 == 0;
    p.out_vec = (uintptr_t)out % (4 * size) == 0 && ld_out % 4 == 0;
    p.v = c->v, p.k_scale = c->k_scale, p.v_scale = c->v_scale;
    p.step = kv_step(*s);
    p.n_pages = c->n_pages, p.n_kv = c->n_kv_head, p.n_seq = s->n_seq, p.D = c->head_dim, p.G = G;
    p.g_inv = (1u << 20) / (unsigned)G + 1u, p.d4_inv = (1u << 20) / (unsigned)(p.D / 4) + 1u;
    p.scale_log2 = scale * 1.44269504088896340736f;
    p.causal = causal, p.window = window, p.err = lm_error_word();

    long long keys = s->max_kv;
    if (window && keys > (long long)window + longest) keys = (long long)window + longest;
    const long long tiles = (keys + PAGE - 1) / PAGE;
    // More than 64 rows: 128 at a time on tcgen05. A batch whose longest sequence has twice the rows of the mean may be a
    // prompt among decode steps: sequences of one token, or of as many rows as the shape for one token holds, go to the
    // kernel for few rows, in a launch of their own.
    const bool many = R > 64, mixed = many && G <= 64 && s->n_seq >= 4 && 2ll * s->n_tok < (long long)s->n_seq * longest;
    const long long rows = !mixed ? R : G <= 8 ? 8 : G <= 16 ? 16 : G <= 32 ? 32 : 64;
    if (many) {
        p.row_min = mixed ? (int)rows : 0;
        if (!launch_kv8_attn_tc(p, c->k, R, tiles)) return false;
        if (!mixed) return true;
        p.row_min = 0;
    }

    // K as [pages x heads x 64, D] bytes; a box is 64 keys of 64 dims, zeros past D
    EncodeFn fn = attn_encode_fn();
    if (!fn) return fail("cuTensorMapEncodeTiled is not available from the driver");
    CUtensorMap map;
    const cuuint64_t dims[2] = { (cuuint64_t)p.D, (cuuint64_t)c->n_pages * c->n_kv_head * PAGE };
    const cuuint64_t strides[1] = { (cuuint64_t)p.D };
    const cuuint32_t box[2] = { 64, PAGE }, estr[2] = { 1, 1 };
    const CUresult r = fn(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void *)c->k, dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail("cuTensorMapEncodeTiled failed (%d) for the K cache", (int)r);

    // Warps of 8 rows (RW = 1) while the rows are few: 8, 16 or 32 rows leave 12, 6 or 3 groups of warps for other tiles.
    // Up to 64 rows: 8 such warps where the device is not filled (17 sequences of 50 rows over a window of 1024: 12.3 us,
    // against 15.0 with 4 warps of 16 rows), else 4 warps of 16 rows, two CTAs an SM (64 sequences of up to 64 rows over 2048
    // tokens, bf16: 131 us against 157).
    const bool big = p.D > 64;
    auto go = [&](auto digits) {
        constexpr int NP = decltype(digits)::value;
        if (rows <= 8) return big ? attn_launch<4, NP, 1, 1, 12, 2, 1>(p, map, tiles) : attn_launch<2, NP, 1, 1, 12, 4, 1>(p, map, tiles);
        if (rows <= 16) return big ? attn_launch<4, NP, 1, 2, 6, 4, 1>(p, map, tiles) : attn_launch<2, NP, 1, 2, 6, 8, 1>(p, map, tiles);
        if (rows <= 32) return big ? attn_launch<4, NP, 1, 4, 3, 6, 1>(p, map, tiles) : attn_launch<2, NP, 1, 4, 3, 8, 1>(p, map, tiles);
        if ((long long)p.n_kv * p.n_seq < ctx().sms)
            return big ? attn_launch<4, NP, 1, 8, 1, 8, 1>(p, map, tiles) : attn_launch<2, NP, 1, 8, 1, 8, 1>(p, map, tiles);
        return big ? attn_launch<4, NP, 2, 4, 1, 6, 2>(p, map, tiles) : attn_launch<2, NP, 2, 4, 1, 8, 2>(p, map, tiles);
    };
    return t == GGML_TYPE_F32 ? go(std::integral_constant<int, 3>()) : go(std::integral_constant<int, 2>());
}
