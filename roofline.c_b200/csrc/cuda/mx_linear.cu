// mx_linear.cu -- tcg_mx_linear: y = x w^T + bias, x in 8 (E4M3) or 4 bits (E2M1), w in 4 bits, a power of two for each 32
// columns of a row, on the tensor core's block-scaled products (tcgen05 kind::mxf8f6f4 and kind::mxf4).
//
//   y[i, n] = sum_b 2^(sx[i, b] + sw[n, b] - 254) sum_{k in block b} cx[i, k] cw[n, k] + bias[n]
//
// Products of codes are exact (at most 6 significant bits), the scales add to the exponent, and the tensor core adds 32 (8
// bits) or 64 columns (4 bits) at a time to an fp32 sum that it cuts after 24 bits; fp32 results are summed in parts of 4096
// columns as far as TMEM holds them. Against 64 bits, normally distributed rows: 5e-8 over 14336 columns in 8 bits (an fp32
// library product on the decoded values: 6e-8), nothing in 4 bits, whose sums fit 24 bits.
//
// The weights are the MMA's first operand: 128 weight rows are TMEM lanes, x's rows columns, so that a warp's 32 lanes hold
// neighbouring results of one row of y and store them as they come, and one token costs 8 columns and not 128 rows.
//   Few rows (mx_stream_kernel): bound by reading the weights. One wave of CTAs, K split over the CTAs of a cluster where the
//     tiles are fewer than the SMs; parts meet in shared memory. One token 4096 -> 14336, x in 8 bits, with weights that
//     are in L2 7.4 us, with weights from DRAM 8.5 (31.2 MB: 3.7 TB/s; ~3.5 us are start, first bytes and end), in 4 bits 6.8
//     and 8.4; 60000 outputs in 4 bits 25 us (5.3 TB/s); 64 rows of 14336 -> 4096 in 8 bits 10.9 and 11.3.
//   Many (mx_pair_kernel): bound by the tensor core and the power that it takes. CTA pairs on tiles of 256 x 256, two
//     accumulators. 4096 rows of 4096 -> 14336 in 4 bits 99 us (4.9 PFLOP/s at ~1.65 GHz: 60% of the cycles; the last round
//     is 8 of 74 pairs' worth), 8192^3 188 us (5.9); 2048 rows of 14336 -> 4096 in 8 bits, fp32 results, 92 us (2.6: two
//     rounds of which the second is three quarters full), 8192^3 358 us (3.1). These are bursts: in a loop of seconds the two
//     prompts take 116 and 108 us under the power cap. (fp32 results: 64 sums a thread in registers, of which 72 bytes spill.)
#include "mx.cuh"
#include "tc05.cuh"

#include <limits.h>
#include <string.h>

#include <atomic>
#include <type_traits>

namespace tcg {
namespace {

constexpr int ERR_WAIT = TCG_ERR_MX_WAIT;
constexpr unsigned long long MX_WAIT_NS = 1000000000ull;    // limit of a wait; the longest, over 2^24 columns, take 0.1 s
constexpr int STREAM_THREADS = 256, MAX_DEPTH = 16, ISSUERS = 2;
constexpr int HALF_SM = 112 * 1024, MOST_SMEM = 226 * 1024;     // of dynamic shared memory; the static part is below 1 KB
constexpr int SUM_K = 4096;             // columns that the tensor core sums before fp32 results are added up outside
constexpr int TILE_N = 128;             // weight rows of a tile: the MMA's M, a TMEM lane each
constexpr int MAX_SPLIT = 8;            // portable cluster size
constexpr int MIN_STAGES = 2;           // of a CTA, where K is split (one token 4096 -> 1024: 3.8 us, with 4 4.4, with 8 4.8)

// What differs between rows in 4 and in 8 bits. A stage is 128 bytes of a row of x; the weights' 4-bit codes next to 8-bit
// rows are spread by the copy itself to 16 bytes for 16 codes, as kind::mxf8f6f4 reads them.
template <int BITS>
struct Fmt {
    static constexpr int K = BITS == 4 ? 256 : 128;         // columns of a stage
    static constexpr int ATOMS = K / MX_ATOM;               // scale groups of a stage
    static constexpr int STEPS = 4;                         // MMAs of a stage: 32 bytes of a row each
    static constexpr int STEP_K = K / STEPS;
    static constexpr uint32_t A_TX = BITS == 4 ? TILE_N * 128 : TILE_N * 64;     // bytes of w that the copy counts
};

// Instruction descriptor: formats (E2M1 is 1 of kind::mxf4, 5 of kind::mxf8f6f4; E4M3 is 0), N / 8 at 17, scales E8M0 at
// 23, M / 128 at 27; the bytes of the scale words that a step takes go to bits 29 (A) and 4 (B).
template <int BITS>
__device__ __forceinline__ uint32_t mx_idesc(int n, int m)
{
    const uint32_t a = BITS == 4 ? 1 : 5, b = BITS == 4 ? 1 : 0;
    return a << 7 | b << 10 | (uint32_t)(n / 8) << 17 | 1u << 23 | (uint32_t)(m / 128) << 27;
}

template <int BITS>
__device__ __forceinline__ void mma_mx(uint32_t d, unsigned long long a, unsigned long long b, uint32_t id, uint32_t sa,
                                       uint32_t sb, uint32_t acc)
{
    if (BITS == 4)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(sa), "r"(sb), "r"(acc));
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(sa), "r"(sb), "r"(acc));
}

// 512 bytes of scales (32 lanes of 16 bytes) to four TMEM columns, the same in each warp's 32 lanes.
__device__ __forceinline__ void scales_to_tmem(uint32_t taddr, uint32_t smem)
{
    const unsigned long long d = (unsigned long long)((smem & 0x3FFFFu) >> 4) | ((unsigned long long)(128 >> 4) << 32) | (1ull << 46);
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(d) : "memory");
}

// One lane of a converged warp. The role loops below run in whole warps and issue under this, so that what they issue is
// known to be the same in all lanes: descriptors then live in uniform registers, where a branch to lane 0 moves each of them
// there (105 cycles a product, which takes 64).
__device__ __forceinline__ bool elect()
{
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}

__device__ __forceinline__ int special_cluster()
{
    int r;
    asm volatile("mov.u32 %0, %%clusterid.x;" : "=r"(r));
    return r;
}
// Bytes from this CTA's shared memory to a peer's, counted by its barrier.
__device__ __forceinline__ void push(uint32_t to, uint32_t from, uint32_t bytes, uint32_t bar)
{
    asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(to), "r"(from), "r"(bytes), "r"(bar) : "memory");
}

struct LinArgs {
    const uint8_t *xs, *ws;             // scales
    const float *bias;
    void *y;
    long long ldy;
    int *err;
    int rows, outs, atoms;              // of x, of w, scale groups of a row
    int stages_k;                       // stages of the whole K
    int tiles_n, tiles_m, split, per;   // CTAs of a tile, stages of each
    unsigned split_inv;                 // 2^16 / split, rounded up
    int tiles, whole;                   // of the pairs: how many, from which on halves
    int acc_stages, accs;               // stages of an accumulator; accumulators of an issuing warp, at most
    int used[2][2];                     // accumulators of the first and the second issuing warp: of a tile's other CTAs, of its last
    int depth;                          // stages in shared memory
    int type;
    bool pairs;                         // two 16-bit results of a row as one word
    int most_loads;                     // stages that a loading warp asks for, at most (tcg_test_mx_withhold_loads)
};

// Wait for the phase of parity `parity`. Gives up when another role has (abort), or MX_WAIT_NS after its first thousand tests
// (bar_wait, tc05.cuh, reads the timer at its start). wait_lane: a warp's lanes may come to differ; they agree again after
// the elected lane has issued what it waited for. wait_for: they agree at once.
__device__ __forceinline__ bool wait_lane(uint32_t bar, uint32_t parity, volatile int *abort, int *err, bool heed_abort = true)
{
    bool here = bar_test(bar, parity);
    unsigned long long since = 0;
    for (uint32_t i = 1; !here; i++) {
        here = bar_test(bar, parity);
        if (!here && (i & 1023) == 0) {
            const unsigned long long now = now_ns();
            if (since == 0) since = now;
            if (now - since > MX_WAIT_NS) {
                *abort = 1;
                atomicExch(err, ERR_WAIT);
                break;
            }
            if (heed_abort && *abort) break;
        }
    }
    return here;
}
__device__ __forceinline__ bool agree(bool ok) { return __all_sync(0xFFFFFFFFu, ok); }
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, volatile int *abort, int *err, bool heed_abort = true)
{
    return agree(wait_lane(bar, parity, abort, err, heed_abort));
}

// N columns of two accumulators, with one wait.
__device__ __forceinline__ void tmem_ld_two(uint32_t at, uint32_t bt, uint32_t (&a)[8], uint32_t (&b)[8])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%16];\n\t"
                 "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%8,%9,%10,%11,%12,%13,%14,%15}, [%17];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]), "=r"(a[4]), "=r"(a[5]), "=r"(a[6]), "=r"(a[7]), "=r"(b[0]),
                   "=r"(b[1]), "=r"(b[2]), "=r"(b[3]), "=r"(b[4]), "=r"(b[5]), "=r"(b[6]), "=r"(b[7])
                 : "r"(at), "r"(bt)
                 : "memory");
}
__device__ __forceinline__ void tmem_ld_two(uint32_t at, uint32_t bt, uint32_t (&a)[16], uint32_t (&b)[16])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%32];\n\t"
                 "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%33];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]), "=r"(a[4]), "=r"(a[5]), "=r"(a[6]), "=r"(a[7]), "=r"(a[8]),
                   "=r"(a[9]), "=r"(a[10]), "=r"(a[11]), "=r"(a[12]), "=r"(a[13]), "=r"(a[14]), "=r"(a[15]), "=r"(b[0]),
                   "=r"(b[1]), "=r"(b[2]), "=r"(b[3]), "=r"(b[4]), "=r"(b[5]), "=r"(b[6]), "=r"(b[7]), "=r"(b[8]), "=r"(b[9]),
                   "=r"(b[10]), "=r"(b[11]), "=r"(b[12]), "=r"(b[13]), "=r"(b[14]), "=r"(b[15])
                 : "r"(at), "r"(bt)
                 : "memory");
}
__device__ __forceinline__ void tmem_ld_two(uint32_t at, uint32_t bt, uint32_t (&a)[32], uint32_t (&b)[32])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%64];\n\t"
                 "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
                 "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%65];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]), "=r"(a[4]), "=r"(a[5]), "=r"(a[6]), "=r"(a[7]), "=r"(a[8]),
                   "=r"(a[9]), "=r"(a[10]), "=r"(a[11]), "=r"(a[12]), "=r"(a[13]), "=r"(a[14]), "=r"(a[15]), "=r"(a[16]),
                   "=r"(a[17]), "=r"(a[18]), "=r"(a[19]), "=r"(a[20]), "=r"(a[21]), "=r"(a[22]), "=r"(a[23]), "=r"(a[24]),
                   "=r"(a[25]), "=r"(a[26]), "=r"(a[27]), "=r"(a[28]), "=r"(a[29]), "=r"(a[30]), "=r"(a[31]), "=r"(b[0]),
                   "=r"(b[1]), "=r"(b[2]), "=r"(b[3]), "=r"(b[4]), "=r"(b[5]), "=r"(b[6]), "=r"(b[7]), "=r"(b[8]), "=r"(b[9]),
                   "=r"(b[10]), "=r"(b[11]), "=r"(b[12]), "=r"(b[13]), "=r"(b[14]), "=r"(b[15]), "=r"(b[16]), "=r"(b[17]),
                   "=r"(b[18]), "=r"(b[19]), "=r"(b[20]), "=r"(b[21]), "=r"(b[22]), "=r"(b[23]), "=r"(b[24]), "=r"(b[25]),
                   "=r"(b[26]), "=r"(b[27]), "=r"(b[28]), "=r"(b[29]), "=r"(b[30]), "=r"(b[31])
                 : "r"(at), "r"(bt)
                 : "memory");
}

// Results of rows row, row + 1 .. of x (as far as there are such rows) for weight row n.
template <int STEP, typename T>
__device__ __forceinline__ void put_columns(const LinArgs &p, int row, int n, float bias, const float (&v)[STEP])
{
    T *y = (T *)p.y + row * p.ldy + n;
    const int rows = n < p.outs ? p.rows - row : 0;
#pragma unroll
    for (int j = 0; j < STEP; j++, y += p.ldy)
        if (j < rows) *y = from_f32<T>(v[j] + bias);
}
// ------------------------------------------------------------------ few rows: K split over clusters

// A stage is 256 columns: 128 bytes of a row in 4 bits, two times 128 next to and in 8 bits. (Four warps that spread the
// weights' codes in shared memory, from boxes of whole 128-byte rows, in place of the copy: one token 4096 -> 14336
// 14.5 us against 10.5.)
template <int BITS, int BN>
struct Stream {
    static constexpr int SUBS = BITS == 8 ? 2 : 1, K = 256, ATOMS = 2;
    static constexpr int A1 = TILE_N * 128, A = SUBS * A1, B1 = BN * 128, B = SUBS * B1, SF = ATOMS * 512;
    static constexpr int STAGE = A + B + 2 * SF;            // every part starts on 1024 bytes
    static constexpr int TX = TILE_N * 128 + B;             // bytes that the copies of codes count: weights as they are held
    static constexpr int COLS = BN <= 32 ? 256 : 512;       // TMEM: accumulators, then the scales
    static constexpr int SF_COLS = 2 * ATOMS * 4, SF_COL = COLS - ISSUERS * SF_COLS;
    static constexpr int MAX_ACC = SF_COL / BN / ISSUERS;   // of an issuing warp
};

// Of a CTA's stages those that the second issuing warp takes: slots are 0 .. depth - 1 in turn, the odd ones are its.
int second_issuer(int stages, int depth)
{
    const int cycles = stages / depth;
    return cycles * (depth / 2) + (stages - cycles * depth) / 2;
}

// One tile of 128 weight rows x BN rows of x a cluster (a tile starts with a group of 128 rows of x, whose scales are four
// TMEM columns: with BN < 128 there is one tile of rows), its K dealt out to the cluster's CTAs. Warp 0 loads, warps 1 and 2
// issue the products, by turns, each on accumulators and scales of its own: what a warp spends on a stage (waiting, copying
// scales, committing: about 500 cycles) is more than the copies need for one (with one issuing warp: one token 4096 ->
// 14336 in 8 bits 8.8 us, with two 7.6; 64 rows of 14336 -> 4096 in 4 bits 9.8 and 9.2). Then all of them take the results.
template <int BITS, int BN>
__global__ void __launch_bounds__(STREAM_THREADS) mx_stream_kernel(const __grid_constant__ CUtensorMap mw, const __grid_constant__ CUtensorMap mx,
                                                                   const __grid_constant__ LinArgs p)
{
    using S = Stream<BITS, BN>;
    extern __shared__ unsigned char raw[];
    __shared__ __align__(8) unsigned long long bars[2 * MAX_DEPTH + 2];
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    unsigned char *const smem = (unsigned char *)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t base = su32(smem), full = su32(bars), empty = full + 8 * MAX_DEPTH, done = empty + 8 * MAX_DEPTH, join = done + 8;
    // a cluster a tile; a division costs as much as a few dozen instructions, so none where there is one tile of rows
    const int rank = (int)cta_rank_in_cluster(), tile = special_cluster(), tm = BN < MX_ATOM ? 0 : tile / p.tiles_n;
    const int n0 = (tile - tm * p.tiles_n) * TILE_N, m0 = tm * BN;
    const int k_begin = rank * p.per, k_end = min(p.stages_k, k_begin + p.per), count = k_end - k_begin;
    // Where a tile's K is split, its results meet by fours of x's rows: the CTA of rank g % split adds up group g.
    const int groups = (min(BN, p.rows - m0) + 3) / 4;
    auto over_split = [&](int i) { return (int)((unsigned)i * p.split_inv >> 16); };        // i / split, of i up to 40
    const int mine = p.split > 1 && groups > rank ? over_split(groups - rank + p.split - 1) : 0;
    if (tid == 0) {
        prefetch_map(&mw), prefetch_map(&mx);
        for (int i = 0; i < p.depth; i++) bar_init(full + 8 * i, 1), bar_init(empty + 8 * i, 1);
        bar_init(done, ISSUERS);
        bar_init(join, 1);
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if (mine) bar_expect_tx(join, (p.split - 1) * mine * TILE_N * 16);
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(&s_tmem)), "r"(S::COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (p.split > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    const uint32_t tmem = s_tmem;
    volatile int *abort = &s_abort;
    bool ok = true;
    pdl_wait();
    lm_signal();
    const int n = n0 + (tid & 127);
    const float bias = p.bias && n < p.outs ? p.bias[n] : 0.0f;
    auto at = [&](int slot) { return base + slot * S::STAGE; };
    auto atoms_of = [&](int k) { return min(S::ATOMS, p.atoms - (k_begin + k) * S::ATOMS); };
    // warp indices as the compiler can see them to be uniform
    const int role = __shfl_sync(0xFFFFFFFFu, warp, 0);
    int loads = 0;
    if (role == 0) {
        const int all = min(count, p.most_loads);
        int slot = 0, phase = 1;
        for (int &k = loads; k < all; k++) {
            const int kk = k_begin + k, na = atoms_of(k);
            ok = wait_lane(empty + 8 * slot, phase, abort, p.err);
            const uint32_t bar = full + 8 * slot, a = at(slot), b = a + S::A, sa = b + S::B, sb = sa + S::SF;
            if (elect() && ok) {
                bar_expect_tx(bar, S::TX + 2 * 512 * na);
#pragma unroll
                for (int i = 0; i < S::SUBS; i++) {
                    tma_load(a + i * S::A1, &mw, bar, (kk * S::SUBS + i) * 128, n0);
                    tma_load(b + i * S::B1, &mx, bar, (kk * S::SUBS + i) * 128, m0);
                }
                bulk_load(sa, p.ws + ((size_t)(n0 / MX_ATOM) * p.atoms + (size_t)kk * S::ATOMS) * 512, 512 * na, bar);
                bulk_load(sb, p.xs + ((size_t)(m0 / MX_ATOM) * p.atoms + (size_t)kk * S::ATOMS) * 512, 512 * na, bar);
            }
            ok = agree(ok);
            if (!ok) break;
            if (++slot == p.depth) slot = 0, phase ^= 1;
        }
    } else if (role <= ISSUERS) {
        const int turn = role - 1;
        const uint32_t id = mx_idesc<BITS>(BN, TILE_N), sfa = tmem + S::SF_COL + turn * S::SF_COLS, sfb = sfa + 4 * S::ATOMS;
        int slot = turn, phase = 0, in_acc = 0;
        uint32_t d = tmem + turn * p.accs * BN;
        // By slots, not by stages: a slot's phases are then waited for by one warp, one after the other. (A warp that waited
        // for a phase while the one before it, another warp's, was still to come would take the one before that for it.)
        for (int k = turn; k < count;) {
            const int na = atoms_of(k);
            ok = wait_lane(full + 8 * slot, phase, abort, p.err);
            fence_after();
            const uint32_t a = at(slot), b = a + S::A, sa = b + S::B, sb = sa + S::SF;
            if (elect() && ok) {
#pragma unroll
                for (int i = 0; i < S::ATOMS; i++)
                    if (i < na) {
                        scales_to_tmem(sfa + 4 * i, sa + 512 * i);
                        scales_to_tmem(sfb + 4 * i, sb + 512 * i);
                    }
#pragma unroll
                for (int j = 0; j < 4 * S::SUBS; j++) {     // 32 bytes of a row each: 64 or 32 columns
                    const int atom = BITS == 8 ? j / 4 : j / 2, byte = BITS == 8 ? j % 4 : j % 2 * 2;
                    const unsigned long long da = sdesc<128>(a + j / 4 * S::A1), db = sdesc<128>(b + j / 4 * S::B1);
                    if (atom < na)
                        mma_mx<BITS>(d, da + 2 * (j % 4), db + 2 * (j % 4), id | byte << 29 | byte << 4, sfa + 4 * atom,
                                     sfb + 4 * atom, in_acc != 0 || j != 0);
                }
                mma_commit(empty + 8 * slot);
            }
            ok = agree(ok);
            if (!ok) break;
            if (slot + ISSUERS < p.depth) slot += ISSUERS, k += ISSUERS;
            else k += p.depth - slot + turn, slot = turn, phase ^= 1;
            if (++in_acc == p.acc_stages) in_acc = 0, d += BN;
        }
        if (elect()) mma_commit(done);
    }
    __syncwarp();
    ok = wait_for(done, 0, abort, p.err, false) && ok && !*abort;
    // After a wait that was given up, copies in flight land before the CTA ends (the one that the loading warp gave up on may
    // have been issued, too).
    if (!ok && role == 0)
        for (int j = max(0, loads - p.depth); j <= min(loads, count - 1); j++)
            wait_for(full + 8 * (j % p.depth), (j / p.depth) & 1, abort, p.err, false);
    fence_after();
    // accumulators that hold something: the first warp's, then the second's
    const int last = rank == p.split - 1, accs0 = p.used[last][0], accs = accs0 + p.used[last][1];
    const uint32_t lane_base = tmem + ((uint32_t)(warp & 3) << 21);
    // Two warps share 32 TMEM lanes (weight rows) and take every second step of columns (x's rows).
    const int t = tid & 127, half = tid >> 7;
    // Before any wait for a peer: a CTA that waits must hold no TMEM that another cluster's CTA on its SM, for which that
    // cluster's other CTAs wait in turn, has asked for.
    auto free_tmem = [&] {
        fence_before();
        __syncthreads();
        if (warp != 0) return;
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::COLS) : "memory");
    };
    auto finish = [&](auto type) {
        using T = decltype(type);
        // [owner][ceil(BN / 4 / split)][128] words of four columns over the stages (whose products are done): what this CTA
        // adds up itself or sends. [sender][..][128] behind the stages: what the cluster's other CTAs send here. (The second
        // over the stages as well leaves room for more of them, but has to wait for the peers' stages: one token 4096 ->
        // 4096 in 4 bits 4.9 us against 4.2.)
        const int per_rank = over_split(BN / 4 + p.split - 1);
        float4 *const sent = (float4 *)smem;
        const float4 *const part = (const float4 *)(smem + p.depth * S::STAGE);
        constexpr int STEP = BN < 32 ? 8 : BN / 2 < 32 ? BN / 2 : 32;
#pragma unroll 1
        for (int c = half * STEP; c < BN && m0 + c < p.rows; c += 2 * STEP) {
            float v[STEP] = {};
            const auto acc = [&](int i) { return lane_base + (i < accs0 ? i : p.accs + i - accs0) * BN + c; };
            for (int i = 0; i < accs; i += 2) {
                uint32_t r[STEP], q[STEP];
                const bool two = i + 1 < accs;
                tmem_ld_two(acc(i), acc(two ? i + 1 : i), r, q);
#pragma unroll
                for (int j = 0; j < STEP; j++) v[j] += __uint_as_float(r[j]);
                if (two)
#pragma unroll
                    for (int j = 0; j < STEP; j++) v[j] += __uint_as_float(q[j]);
            }
            if (p.split > 1) {
#pragma unroll
                for (int j = 0; j < STEP; j += 4) {
                    const int g = (c + j) / 4, i = over_split(g), owner = g - i * p.split;
                    sent[(owner * per_rank + i) * TILE_N + t] = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                }
            } else if (ok) {
                put_columns<STEP, T>(p, m0 + c, n, bias, v);
            }
        }
        if (p.split > 1) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        free_tmem();
        if (p.split == 1) return;
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");     // the peers' barriers are there
        const int to = tid - 128;                       // not by warp 0, which gives the TMEM back meanwhile
        if (to >= 0 && to < p.split && to < groups && to != rank)
            push(peer_addr(su32(part + (rank - (rank > to)) * per_rank * TILE_N), to), su32(sent + to * per_rank * TILE_N),
                 over_split(groups - to + p.split - 1) * TILE_N * 16, peer_addr(join, to));
        __syncwarp();
        const bool came = !mine || wait_for(join, 0, abort, p.err, false);
        ok = ok && came;
        asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
#pragma unroll 2
        for (int i = half; i < mine; i += 2) {
            float sum[4] = {};
#pragma unroll
            for (int s = 0; s < MAX_SPLIT; s++) {
                if (s == 4 && p.split <= 4) break;          // one branch; the parts before it are loaded together
                const float4 *const from = s == rank ? sent + rank * per_rank * TILE_N : part + (s - (s > rank)) * per_rank * TILE_N;
                const float4 v = s < p.split ? from[i * TILE_N + t] : make_float4(0, 0, 0, 0);
                sum[0] += v.x, sum[1] += v.y, sum[2] += v.z, sum[3] += v.w;
            }
            if (ok) put_columns<4, T>(p, m0 + 4 * (rank + i * p.split), n, bias, sum);
        }
        // A CTA leaves when all that it sent has arrived: when every CTA of the cluster has received.
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        if (!came) wait_for(join, 0, abort, p.err, false);      // sent late, but sent by now
    };
    if (p.type == GGML_TYPE_F32) finish(float());
    else if (p.type == GGML_TYPE_F16) finish(__half());
    else finish(__nv_bfloat16());
}

// ------------------------------------------------------------------ many rows: CTA pairs

// A cluster of two CTAs computes tiles of 256 weight rows x 256 rows of x, one after the other: CTA r holds weight rows
// 128 r .. 128 r + 127 (in its shared memory, and as the lanes of its accumulators) and half of x's rows; the pair's
// products read both halves. Each CTA has the scales of its weight rows and of all 256 rows of x.
template <int BITS>
struct Pair {
    static constexpr int ROWS = 256;                        // of x
    static constexpr int A = TILE_N * 128, B = ROWS / 2 * 128, SF = Fmt<BITS>::ATOMS * 512;
    static constexpr int STAGE = (A + B + 3 * SF + 1023) / 1024 * 1024;
    static constexpr int STAGES = 6;
    static constexpr uint32_t TX = 2 * (Fmt<BITS>::A_TX + B + 3 * SF);
    // Two accumulators of 256 columns and the scales do not fit 512 columns; the second starts 32 columns before the first
    // one's end. Those 32 are drained before anything else, so the next tile's products wait for an eighth of a drain.
    static constexpr int ACC1 = 224, SF_COL = 480, COLS = 512;
    static constexpr int SMEM = 1024 + STAGES * STAGE;
    static_assert(SF_COL + 3 * 4 * Fmt<BITS>::ATOMS <= COLS, "the scales fit behind the accumulators");
};

constexpr int PAIR_EPI = 16, PAIR_THREADS = 32 * (2 + PAIR_EPI);

template <int BITS>
__device__ __forceinline__ void mma_mx_pair(uint32_t d, unsigned long long a, unsigned long long b, uint32_t id, uint32_t sa,
                                            uint32_t sb, uint32_t acc)
{
    if (BITS == 4)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(sa), "r"(sb), "r"(acc));
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(sa), "r"(sb), "r"(acc));
}
__device__ __forceinline__ void scales_to_tmem_pair(uint32_t taddr, uint32_t smem)
{
    const unsigned long long d = (unsigned long long)((smem & 0x3FFFFu) >> 4) | ((unsigned long long)(128 >> 4) << 32) | (1ull << 46);
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(d) : "memory");
}
// The pair's products so far, to the barrier at this offset in both CTAs.
__device__ __forceinline__ void commit_pair(uint32_t bar)
{
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(bar), "h"((unsigned short)3) : "memory");
}

// The i-th tile, in the order they are taken: eight blocks of x's rows at a time, so that the tiles under way together share
// both operands. What is left for the last round goes by halves of 128 rows of x where each pair gets at most one.
struct PairTile {
    int n0, m0, rows;                                       // first weight row, first row of x, 256 or 128 of them
};
__device__ __forceinline__ PairTile tile_at(const LinArgs &p, int i)
{
    const bool half = i >= p.whole;
    if (half) i -= p.whole;
    const int tile = half ? p.whole + i / 2 : i;
    const int group = tile / (8 * p.tiles_n), in = tile - group * 8 * p.tiles_n, high = min(8, p.tiles_m - 8 * group);
    const int tn = in / high, tm = 8 * group + in - tn * high;
    return { tn * 256, tm * 256 + (half ? i % 2 * 128 : 0), half ? 128 : 256 };
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b)
{
    const T v[2] = { from_f32<T>(a), from_f32<T>(b) };
    uint32_t w;
    memcpy(&w, v, sizeof w);
    return w;
}

template <typename T, int BITS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PAIR_THREADS, 1)
mx_pair_kernel(const __grid_constant__ CUtensorMap mw, const __grid_constant__ CUtensorMap mx, const __grid_constant__ CUtensorMap msw,
               const __grid_constant__ CUtensorMap msx, const __grid_constant__ LinArgs p)
{
    using F = Fmt<BITS>;
    using S = Pair<BITS>;
    extern __shared__ unsigned char raw[];
    // full, empty a stage; full, free, overlap free an accumulator; the end
    __shared__ __align__(8) unsigned long long bars[2 * S::STAGES + 7];
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    const uint32_t base = (su32(raw) + 1023) & ~1023u;
    const int tid = threadIdx.x, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0), lane = tid & 31;
    const uint32_t rank = blockIdx.x & 1;
    const uint32_t full = su32(bars), empty = full + 8 * S::STAGES, acc_full = empty + 8 * S::STAGES, acc_free = acc_full + 16,
                   lap_free = acc_free + 16, end = lap_free + 16;
    if (tid == 0) {
        prefetch_map(&mw), prefetch_map(&mx), prefetch_map(&msw), prefetch_map(&msx);
        for (int i = 0; i < S::STAGES; i++) bar_init(full + 8 * i, 1), bar_init(empty + 8 * i, 1);
        for (int i = 0; i < 2; i++) {
            bar_init(acc_full + 8 * i, 1);
            bar_init(acc_free + 8 * i, 2 * PAIR_EPI);       // every draining warp of both CTAs
            bar_init(lap_free + 8 * i, 8);                  // those that hold the shared columns
        }
        bar_init(end, 1);
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(&s_tmem)), "r"(S::COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    cluster_sync();                                         // barriers and TMEM are there in both CTAs
    fence_after();
    const uint32_t tmem = s_tmem;
    volatile int *abort = &s_abort;
    bool ok = true;
    pdl_wait();
    const int first = blockIdx.x >> 1, step = gridDim.x >> 1;
    // Units: a tile's K, or with F32 results a part of it at a time.
    if (warp == 0) {
        int slot = 0, phase = 1, issued = 0;
        for (int tile = first; tile < p.tiles && ok; tile += step) {
            const PairTile at = tile_at(p, tile);
            const int n0 = at.n0 + rank * 128, m0 = at.m0, mine = m0 + rank * (at.rows / 2);    // a half's box brings 64 rows too many
            for (int k = 0; k < p.stages_k && issued < p.most_loads; k++) {
                ok = wait_lane(empty + 8 * slot, phase, abort, p.err);
                const uint32_t a = base + slot * S::STAGE, b = a + S::A, sa = b + S::B, sb = sa + S::SF;
                const uint32_t bar = peer_addr(full + 8 * slot, 0);
                if (elect() && ok) {
                    if (rank == 0) bar_expect_tx(full + 8 * slot, S::TX);
                    tma_load_pair(a, &mw, bar, k * 128, n0);
                    tma_load_pair(b, &mx, bar, k * 128, mine);
                    tma_load_pair(sa, &msw, bar, k * (F::ATOMS * 64), n0 / 128);
                    tma_load_pair(sb, &msx, bar, k * (F::ATOMS * 64), m0 / 128);
                }
                ok = agree(ok);
                issued++;                                   // or perhaps not, where it gave up
                if (++slot == S::STAGES) slot = 0, phase ^= 1;
                if (!ok) break;
            }
        }
        // copies in flight land before the CTAs end (both CTAs' complete on the leader's barriers)
        if (rank == 0)
            for (int i = 1; i <= S::STAGES && i <= issued; i++) {
                const int at = slot - i, wrapped = at < 0;
                wait_for(full + 8 * (wrapped ? at + S::STAGES : at), phase ^ 1 ^ wrapped, abort, p.err, false);
            }
    } else if (warp == 1 && rank == 0) {
        const uint32_t sfa = tmem + S::SF_COL, sfb = sfa + 4 * F::ATOMS;
        int slot = 0, phase = 0;
        uint32_t unit = 0;
        for (int tile = first; tile < p.tiles && ok; tile += step) {
            const uint32_t id = mx_idesc<BITS>(tile_at(p, tile).rows, 256);
            for (int k0 = 0; k0 < p.stages_k && ok; k0 += p.acc_stages, unit++) {
                const uint32_t buf = unit & 1, d = tmem + (buf ? S::ACC1 : 0);
                ok = wait_for(acc_free + 8 * buf, (unit >> 1 & 1) ^ 1, abort, p.err) &&
                     (unit == 0 || wait_for(lap_free + 8 * (buf ^ 1), (unit - 1) >> 1 & 1, abort, p.err));
                fence_after();
                const int k1 = min(p.stages_k, k0 + p.acc_stages);
                for (int k = k0; k < k1 && ok; k++) {
                    const int na = min(F::ATOMS, p.atoms - k * F::ATOMS);
                    ok = wait_lane(full + 8 * slot, phase, abort, p.err);
                    fence_after();
                    const uint32_t a = base + slot * S::STAGE, b = a + S::A, sa = b + S::B, sb = sa + S::SF;
                    if (elect() && ok) {
#pragma unroll
                        for (int i = 0; i < F::ATOMS; i++) {
                            scales_to_tmem_pair(sfa + 4 * i, sa + 512 * i);
                            scales_to_tmem_pair(sfb + 8 * i, sb + 512 * i);
                            scales_to_tmem_pair(sfb + 8 * i + 4, sb + S::SF + 512 * i);
                        }
                        const unsigned long long da = sdesc<128>(a), db = sdesc<128>(b);
#pragma unroll
                        for (int j = 0; j < F::STEPS; j++) {
                            const int atom = j * F::STEP_K / MX_ATOM, byte = j * F::STEP_K / MX_BLOCK % 4;
                            if (atom < na)
                                mma_mx_pair<BITS>(d, da + 2 * j, db + 2 * j, id | byte << 29 | byte << 4, sfa + 4 * atom,
                                                  sfb + 8 * atom, k != k0 || j != 0);
                        }
                        commit_pair(empty + 8 * slot);
                    }
                    ok = agree(ok);
                    if (!ok) break;
                    if (++slot == S::STAGES) slot = 0, phase ^= 1;
                }
                if (ok && elect()) commit_pair(acc_full + 8 * buf);
                __syncwarp();
            }
        }
        // the other CTA's roles leave, too
        if (!ok && elect()) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(peer_addr(su32(&s_abort), 1)), "r"(1) : "memory");
        // every product issued above has ended once this flips
        if (elect())
            asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(end) : "memory");
        __syncwarp();
        wait_for(end, 0, abort, p.err, false);
    } else if (warp >= 2) {
        const int q = warp & 3, h = (warp - 2) >> 2;        // TMEM lanes 32 q .., columns 64 h ..
        const uint32_t at = tmem + ((uint32_t)q << 21) + 64 * h;
        const uint32_t free_bar = peer_addr(acc_free, 0), lap_bar = peer_addr(lap_free, 0);
        uint32_t unit = 0;
        for (int tile = first; tile < p.tiles && ok; tile += step) {
            const int n = tile_at(p, tile).n0 + rank * 128 + 32 * q + lane;
            // the order of 16-column pieces: the shared columns are the last 32 of the first accumulator, the first of the second
            auto piece = [&](int i) { return (i ^ (h == 3 ? 2 : 0)) * 16; };
            const float bias = p.bias && n < p.outs ? p.bias[n] : 0.0f;
            // 64 columns: fp32 results are summed here over the tile's units; 16-bit ones have one unit and are packed at once
            constexpr bool WIDE = sizeof(T) == 4;
            constexpr int WORDS = WIDE ? 16 : 8;            // of 16 columns
            uint32_t acc[4][WORDS];
            if (WIDE)
#pragma unroll
                for (int i = 0; i < 4 * WORDS; i++) acc[i / WORDS][i % WORDS] = __float_as_uint(bias);
            for (int k0 = 0; k0 < p.stages_k; k0 += p.acc_stages, unit++) {
                const uint32_t buf = unit & 1;
                ok = wait_for(acc_full + 8 * buf, unit >> 1 & 1, abort, p.err);
                if (!ok) break;
                fence_after();
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    uint32_t r[16];
                    tmem_ld16(at + (buf ? S::ACC1 : 0) + piece(i), r);
#pragma unroll
                    for (int j = 0; j < 16; j += WIDE ? 1 : 2) {
                        if constexpr (WIDE) acc[i][j] = __float_as_uint(__uint_as_float(acc[i][j]) + __uint_as_float(r[j]));
                        else acc[i][j / 2] = pack2<T>(__uint_as_float(r[j]) + bias, __uint_as_float(r[j + 1]) + bias);
                    }
                    if (i == 1) {                           // the shared columns are drained
                        fence_before();
                        __syncwarp();
                        if (h == (buf ? 0 : 3) && lane == 0) bar_arrive_cluster(lap_bar + 8 * buf);
                    }
                }
                fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive_cluster(free_bar + 8 * buf);
            }
            if (!ok) break;
            int again = tile;                               // taken anew: the registers are the accumulators' until here
            asm volatile("" : "+r"(again));
            const PairTile here = tile_at(p, again);
            const int m0 = here.m0 + 64 * h, end = min(p.rows, here.m0 + here.rows);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int m = m0 + piece(i), rows = n < p.outs ? end - m : 0;
                if constexpr (WIDE) {
                    T *y = (T *)p.y + m * p.ldy + n;
#pragma unroll
                    for (int j = 0; j < 16; j++, y += p.ldy)
                        if (j < rows) *y = __uint_as_float(acc[i][j]);
                } else if (p.pairs) {
                    // a lane trades with its neighbour: two features of one row instead of one feature of two
                    T *y = (T *)p.y + (m + (lane & 1)) * p.ldy + (n & ~1);
#pragma unroll
                    for (int j = 0; j < 8; j++, y += 2 * p.ldy) {
                        const uint32_t own = acc[i][j], other = __shfl_xor_sync(0xFFFFFFFFu, own, 1);
                        if (2 * j + (lane & 1) < rows)
                            *(uint32_t *)y = lane & 1 ? __byte_perm(other, own, 0x7632) : __byte_perm(own, other, 0x5410);
                    }
                } else {
                    unsigned short *y = (unsigned short *)p.y + m * p.ldy + n;
#pragma unroll
                    for (int j = 0; j < 16; j++, y += p.ldy)
                        if (j < rows) *y = (unsigned short)(acc[i][j / 2] >> (j & 1) * 16);
                }
            }
        }
    }
    fence_before();
    __syncthreads();
    cluster_sync();                                         // the leader's products into this CTA's TMEM have ended
    if (warp == 1) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::COLS) : "memory");
    }
}

// ------------------------------------------------------------------ launch

// Boxes of 128 bytes of shared memory x box_rows in the 128-byte swizzle. spread: 4-bit codes, 16 of them to 16 bytes.
bool encode_mx(CUtensorMap *map, const tcg_mx_t &m, int box_rows, bool spread)
{
    const EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return fail("cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t pitch = (cuuint64_t)mx_pitch(m.cols, m.bits);
    cuuint64_t dims[2] = { spread ? (cuuint64_t)mx_wide(m.cols) : pitch, (cuuint64_t)m.rows };
    cuuint64_t strides[1] = { pitch };
    cuuint32_t box[2] = { 128, (cuuint32_t)box_rows };
    cuuint32_t estr[2] = { 1, 1 };
    const CUresult r = fn(map, spread ? CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B : CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void *)m.codes,
                          dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail("cuTensorMapEncodeTiled failed (%d) for [%d x %d] in %d bits", (int)r, m.rows, m.cols, m.bits);
    return true;
}

// The scales as rows of 64-bit words, a row for each 128 rows of the matrix; boxes of a stage's scales of `blocks` rows.
bool encode_scales(CUtensorMap *map, const tcg_mx_t &m, int atoms, int blocks)
{
    const EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return fail("cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t wide = (cuuint64_t)mx_wide(m.cols) / MX_ATOM * 64;
    cuuint64_t dims[2] = { wide, ((cuuint64_t)m.rows + MX_ATOM - 1) / MX_ATOM };
    cuuint64_t strides[1] = { wide * 8 };
    cuuint32_t box[2] = { (cuuint32_t)atoms * 64, (cuuint32_t)blocks };
    cuuint32_t estr[2] = { 1, 1 };
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT64, 2, (void *)m.scales, dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail("cuTensorMapEncodeTiled failed (%d) for the scales of [%d x %d]", (int)r, m.rows, m.cols);
    return true;
}

// The shared memory that a kernel may ask for, set at its first call on each device. (Calls that come first together set the
// same.)
template <auto FN>
bool allow_smem(int bytes)
{
    static std::atomic<bool> done[64];
    std::atomic<bool> &here = done[ctx().device & 63];
    if (here.load(std::memory_order_acquire)) return true;
    TCG_CUDA(cudaFuncSetAttribute(FN, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    here.store(true, std::memory_order_release);
    return true;
}

template <typename T, int BITS>
bool pair_launch(LinArgs &p, const tcg_mx_t &x, const tcg_mx_t &w)
{
    using S = Pair<BITS>;
    using F = Fmt<BITS>;
    CUtensorMap mw, mx, msw, msx;
    if (!encode_mx(&mw, w, TILE_N, BITS == 8) || !encode_mx(&mx, x, S::ROWS / 2, false) ||
        !encode_scales(&msw, w, F::ATOMS, 1) || !encode_scales(&msx, x, F::ATOMS, 2))
        return false;
    p.tiles_n = (p.outs + 255) / 256;
    p.tiles_m = (p.rows + S::ROWS - 1) / S::ROWS;
    p.stages_k = (p.atoms + F::ATOMS - 1) / F::ATOMS;
    p.pairs = p.ldy % 2 == 0 && (uintptr_t)p.y % 4 == 0 && p.outs % 2 == 0;
    p.acc_stages = sizeof(T) == 4 ? SUM_K / F::K : p.stages_k;
    const long long tiles = (long long)p.tiles_n * p.tiles_m, most = ctx().sms / 2;
    if (tiles > 0x7fffff00ll) return fail("tcg_mx_linear: %d rows and %d outputs are too many for one call", p.rows, p.outs);
    const int left = (int)(tiles % most);
    const bool halve = 2 * left <= most;
    p.whole = (int)(halve ? tiles - left : tiles);
    p.tiles = p.whole + (halve ? 2 * left : 0);
    const int pairs = (int)min((long long)p.tiles, most);
    constexpr auto fn = mx_pair_kernel<T, BITS>;
    if (!allow_smem<fn>(S::SMEM)) return false;
    TCG_CUDA(launch_pdl(fn, dim3(2 * pairs), dim3(PAIR_THREADS), S::SMEM, ctx().cur, mw, mx, msw, msx, (const LinArgs)p));
    return true;
}

// What a call takes, estimated in ns from B200 measurements, to choose between the kernels and the number of parts of K:
//   rows, columns -> outputs, bits     stream (us)                         pair
//   1, 14336 -> 4096, 8                13.9, 4 parts 7.2
//   64, 4096 -> 4096, 4                6.4, 2 parts 6.8, 4 parts 6.8
//   128, 14336 -> 4096, 8              24.2, 2 parts 22.5, 4 parts 15.8    25.6
//   512, 4096 -> 4096, 4               8.2                                 10.0
//   300, 14336 -> 4096, 8              31.0                                29.2
//   200, 4096 -> 14336, 8              23.2                                17.4
//   1000, 4096 -> 4096, 4              15.8                                11.9
// A CTA of the stream kernel starts and ends in 3 us and 11 ns a row of x's tile; a stage of 256 columns takes what its MMAs
// and waits take, and more the more CTAs read; the join of parts takes 600 ns and 20 a row, and with 128 rows in 8 bits
// leaves room for only two stages in flight.
template <int BITS, int BN>
double stream_ns(int rows, long long tiles, int stages, int split)
{
    const double waves = (double)((tiles * split + ctx().sms - 1) / ctx().sms), r = min(BN, rows);
    const double stage = (BITS == 4 ? 165 : BN <= 64 ? 220 : split == 1 ? 340 : 440)
        + (double)min(tiles * split, (long long)ctx().sms) * Stream<BITS, BN>::STAGE * 1.8e-5;
    return waves * (3000 + 11 * r + (stages + split - 1) / split * stage) + (split > 1 ? 600 + 20 * r : 0);
}

// Clusters of `split` CTAs that run at once on this thread's device. Those of eight with an SM's shared memory each are 15 on a
// B200, not 148 / 8: 16 of them take two rounds (200 rows of 4096 -> 1024 in 8 bits in eight parts 13.1 us, in five 9.1). 0
// after an error.
template <int BITS, int BN>
int clusters_at_once(int split)
{
    static std::atomic<int> of_device[64][MAX_SPLIT + 1];
    std::atomic<int> &known = of_device[ctx().device & 63][split];
    int n = known.load(std::memory_order_relaxed);
    if (n) return n;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = { (unsigned)split, 1, 1 };
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)split);
    lc.blockDim = dim3(STREAM_THREADS);
    lc.dynamicSmemBytes = MOST_SMEM;
    lc.attrs = &attr;
    lc.numAttrs = 1;
    constexpr auto fn = mx_stream_kernel<BITS, BN>;
    if (!allow_smem<fn>(MOST_SMEM)) return 0;
    if (cudaOccupancyMaxActiveClusters(&n, fn, &lc) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    known.store(n, std::memory_order_relaxed);
    return n;
}

struct StreamPlan {
    int split;
    double ns;
};
template <int BITS, int BN>
StreamPlan stream_plan(int rows, long long tiles, int stages)
{
    StreamPlan best = { 1, stream_ns<BITS, BN>(rows, tiles, stages, 1) };
    for (int s = 2; s <= MAX_SPLIT && tiles * s <= ctx().sms && s * MIN_STAGES <= stages; s++) {
        const double ns = stream_ns<BITS, BN>(rows, tiles, stages, s);
        if (ns < best.ns && tiles <= clusters_at_once<BITS, BN>(s)) best = { s, ns };
    }
    return best;
}

// Rounds of the pairs; the last one's tiles are halved where each pair gets at most one half.
template <int BITS>
double pair_ns(long long tiles, int stages)
{
    const long long pairs = ctx().sms / 2, left = tiles % pairs;
    const double round = 2100 + stages * (BITS == 4 ? 290 : 590), last = 2400 + stages * (BITS == 4 ? 240 : 400);
    return 3700 + (double)(tiles / pairs) * round + (left == 0 ? 0 : 2 * left <= pairs ? min(last, round) : round);
}

template <int BITS, int BN>
bool stream_launch(LinArgs &p, const tcg_mx_t &x, const tcg_mx_t &w)
{
    using S = Stream<BITS, BN>;
    if (BN < MX_ATOM && p.rows > BN) return fail("tcg_mx_linear: %d rows in tiles of %d", p.rows, BN);
    CUtensorMap mw, mx;
    if (!encode_mx(&mw, w, TILE_N, BITS == 8) || !encode_mx(&mx, x, BN, false)) return false;
    p.tiles_n = (p.outs + TILE_N - 1) / TILE_N;
    p.stages_k = (p.atoms + S::ATOMS - 1) / S::ATOMS;
    const long long tiles = (long long)p.tiles_n * ((p.rows + BN - 1) / BN);
    p.split = stream_plan<BITS, BN>(p.rows, tiles, p.stages_k).split;
    p.per = (p.stages_k + p.split - 1) / p.split;
    p.split = (p.stages_k + p.per - 1) / p.per;
    // Half an SM's shared memory a CTA: undivided, one wave leaves room for the next kernel's CTAs to start in (one token
    // 4096 -> 14336 in 4 bits 6.8 us, with all of it 7.6), several waves run two CTAs an SM (60000 outputs 25 us, with one
    // CTA 31). Not where one wave would have fewer than four stages (4096 -> 14336 in 8 bits 7.5 us, with half 9.1) or K is
    // split (14336 -> 4096 in 4 bits 7.0 us, with half 7.3).
    const bool half = BN <= 32 && (tiles * p.split > ctx().sms || (p.split == 1 && 4 * S::STAGE + 16 * 1024 <= HALF_SM));
    const int room = (half ? HALF_SM : MOST_SMEM) - 1024;
    p.split_inv = (65536 + p.split - 1) / p.split;
    const int part = p.split > 1 ? (p.split - 1) * ((BN / 4 + p.split - 1) / p.split) * TILE_N * 16 : 0;
    p.depth = min(MAX_DEPTH, min(max(p.per, 2), (room - part) / S::STAGE));
    const size_t smem = 1024 + p.depth * S::STAGE + part;
    // fp32 results: accumulators of SUM_K columns, or as many as TMEM holds
    const int own = p.per - second_issuer(p.per, p.depth);  // stages of the first issuing warp, which has more
    p.acc_stages = p.type == GGML_TYPE_F32 ? max((own + S::MAX_ACC - 1) / S::MAX_ACC, SUM_K / S::K) : own;
    p.accs = (own + p.acc_stages - 1) / p.acc_stages;
    for (int last = 0; last < 2; last++) {
        const int count = last ? p.stages_k - (p.split - 1) * p.per : p.per, second = second_issuer(count, p.depth);
        p.used[last][0] = (count - second + p.acc_stages - 1) / p.acc_stages;
        p.used[last][1] = (second + p.acc_stages - 1) / p.acc_stages;
    }
    if (tiles * p.split > 0x7fffffffll) return fail("tcg_mx_linear: %d rows and %d outputs are too many for one call", p.rows, p.outs);
    constexpr auto fn = mx_stream_kernel<BITS, BN>;
    if (!allow_smem<fn>(MOST_SMEM)) return false;
    cudaLaunchAttribute attrs[2];
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)(tiles * p.split));
    lc.blockDim = dim3(STREAM_THREADS);
    lc.dynamicSmemBytes = smem;
    lc.stream = ctx().cur;
    lc.attrs = attrs;
    lc.numAttrs = pdl_attr(attrs);
    attrs[lc.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attrs[lc.numAttrs].val.clusterDim = { (unsigned)p.split, 1, 1 };
    lc.numAttrs++;
    TCG_CUDA(cudaLaunchKernelEx(&lc, fn, mw, mx, (const LinArgs)p));
    return true;
}

template <int BITS>
bool linear_go(LinArgs &p, const tcg_mx_t &x, const tcg_mx_t &w)
{
    if (p.rows <= 8) return stream_launch<BITS, 8>(p, x, w);
    if (p.rows <= 16) return stream_launch<BITS, 16>(p, x, w);
    if (p.rows <= 32) return stream_launch<BITS, 32>(p, x, w);
    if (p.rows <= 64) return stream_launch<BITS, 64>(p, x, w);
    const int stages = (p.atoms + 1) / 2;
    const long long wide = (long long)((p.rows + 255) / 256) * ((p.outs + 255) / 256);
    const long long tiles = (long long)((p.rows + 127) / 128) * ((p.outs + 127) / 128);
    if (pair_ns<BITS>(wide, stages) < stream_plan<BITS, 128>(p.rows, tiles, stages).ns)
        return lm_by_type((ggml_type_t)p.type, [&](auto v) { return pair_launch<decltype(v), BITS>(p, x, w); });
    return stream_launch<BITS, 128>(p, x, w);
}

std::atomic<int> g_most_loads{INT_MAX};

}  // namespace
}  // namespace tcg

using namespace tcg;

// Test hook for the paths of a wait that gives up: with stages >= 0, the loading warps of the calls after it (of every
// thread) ask for that many stages and no more, so that the waits for the next one run out; a negative number restores
// normal operation. Returns the number before.
extern "C" int tcg_test_mx_withhold_loads(int stages)
{
    const int before = g_most_loads.exchange(stages < 0 ? INT_MAX : stages);
    return before == INT_MAX ? -1 : before;
}

extern "C" bool tcg_mx_linear(void *y, const tcg_mx_t *x, const tcg_mx_t *w, const float *bias, int64_t ld_y, ggml_type_t t)
{
    const char *who = "tcg_mx_linear";
    if (!lm_type_size(t)) return fail("%s: type %d is not F32, F16 or BF16", who, (int)t);
    if (!mx_check(who, "x", x) || !mx_check(who, "w", w)) return false;
    if (w->bits != 4) return fail("%s: weights in %d bits: 4", who, w->bits);
    if (x->cols != w->cols) return fail("%s: rows of %d columns and weights of %d", who, x->cols, w->cols);
    if (w->rows && !mx_rows(who, "y", y, x->rows, w->rows, ld_y, t)) return false;
    if ((uintptr_t)bias % 4) return fail("%s: misaligned bias", who);
    if (!lm_ready(who)) return false;
    if (!x->rows || !w->rows) return true;
    LinArgs p = {};
    p.xs = x->scales, p.ws = w->scales, p.bias = bias, p.y = y, p.ldy = ld_y, p.err = lm_error_word();
    p.most_loads = g_most_loads;
    p.rows = x->rows, p.outs = w->rows, p.atoms = (int)(mx_wide(x->cols) / MX_ATOM), p.type = t;
    return x->bits == 4 ? linear_go<4>(p, *x, *w) : linear_go<8>(p, *x, *w);
}
