// Paged multi-query attention for decode and speculative verification over a 4-bit KV cache:
// the call of nanovllm/layers/attention.py:71-74 on records of kv_q4.cuh.
//
// Work decomposition, scheduling, split-K merge and the bounded waits are those of
// paged_attention.cu (paged_plan.cuh); a stage is 128 records of keys and 128 of values, two
// contiguous 10 KiB bulk copies.
//
// Mathematics.  A cached value is s n + m with n the 4-bit code and one (s, m) per group of 32
// head dimensions, so per query row and token
//     q . k = sum_g ( s_g (q_g . n_g) + m_g sum(q_g) ),      o_g = sum_t (p_t s_tg) n_tg + sum_t p_t m_tg.
// The codes themselves are the matrix operands: a nibble in the low bits of an fp16 lane is the
// subnormal n * 2^-24 (16 n * 2^-24 one nibble up), exactly, so that a mask turns a word of
// codes into operands of mma.sync.m16n8k16 and nothing is converted.  The powers of two are
// undone in fp32; the queries that meet the second nibble carry a factor 1/16.  Scales and
// minima are applied in fp32 on the results (keys) and on the probabilities (values); p s is
// rounded to fp16 (2^-12 relative), q is exact in fp16 after scaling each row by a power of two.
//
// As in the 16-bit kernel's transposed form tokens are the M of the matrix products and query
// rows their N (8 per tile, NT tiles): S^T = K Q^T, O^T += V^T (P s)^T.  ldmatrix hands lane
// (g, c) word c of token g's four groups; its transposed form hands it half-word g of tokens
// 2 c and 2 c + 1, again one nibble per token in either half of a register.
//
// Ranges.  A row's probabilities are 2^(x - r) with r = (lazy running maximum) + E, where 2^E
// follows the largest value scale the warp has met (raised when a scale exceeds 2^7 times it):
// p s then stays below 2^15 and small scales do not underflow fp16.
#include <cfloat>
#include <climits>

#include "kv_q4.cuh"
#include "paged_plan.cuh"

namespace b200 {
namespace pa {
namespace {

using q4::hi_f;
using q4::kGroups;
using q4::kRecord;
using q4::lo_f;

constexpr int kKvBytes = kTile * kRecord;  // keys (or values) of one stage
constexpr int kStage = 2 * kKvBytes;
constexpr int32_t kNoPage = 4;             // header flag: the tile's block id is not in the cache
constexpr float kNone = -1e30f;            // reference of a row that has met no token
constexpr int kExpMin = -60, kExpMax = 60; // bounds of E and of the query rows' exponents

struct Q4Params {
    Params base;
    const uint8_t* k;
    const uint8_t* v;
};

template <int NT>
struct Cfg {
    // Up to 8 query rows: two CTAs per SM, one of them computes while the other waits or combines.
    static constexpr int kCtas = NT == 1 ? 2 : 1;
    static constexpr int kStages = NT == 1 ? 4 : 7;
};

template <int NT>
struct Smem {
    alignas(128) uint8_t stages[Cfg<NT>::kStages][kStage];
    uint8_t qbuf[Cfg<NT>::kStages][8 * NT * kD * 2];
    float co[kConsumerWarps / 2][8 * NT][kD];
    float cm[kConsumerWarps][8 * NT];
    float cl[kConsumerWarps][8 * NT];
    Header hdr[Cfg<NT>::kStages];
    uint64_t full[Cfg<NT>::kStages];
    uint64_t empty[Cfg<NT>::kStages];
    uint64_t cbar;
    int32_t off[kMaxBatch + 1];
    int32_t red[kThreads / 32 + 1];
    int32_t flag;
    int32_t err;
};
static_assert(sizeof(Smem<1>) <= 233472 / 2 - 1024 && sizeof(Smem<2>) <= 232448, "shared memory over the SM's");

__device__ __forceinline__ void bulk_load_hint(void* dst, const void* src, uint32_t bytes, uint64_t* bar,
                                               uint64_t policy) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(
            smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_u32(bar)), "l"(policy)
        : "memory");
}

__device__ __forceinline__ float exp2_int(int e) { return __int_as_float((127 + e) << 23); }  // -126 <= e <= 127

template <bool BF16, int NT>
__global__ void __launch_bounds__(kThreads, Cfg<NT>::kCtas) paged_attention_q4_kernel(const __grid_constant__ Q4Params qp) {
    constexpr int NS = Cfg<NT>::kStages;
    const Params& p = qp.base;
    extern __shared__ uint8_t smem_raw[];
    Smem<NT>& sm = *reinterpret_cast<Smem<NT>*>(smem_raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        for (int s = 0; s < NS; ++s) {
            mbar_init(&sm.full[s], 1);
            mbar_init(&sm.empty[s], kConsumerWarps);
        }
        mbar_init(&sm.cbar, kConsumers);
        sm.err = 0;
        fence_mbar_init();
    }
    // The producer's first claim does not depend on the plan: its latency overlaps the planning.
    const bool producer = warp == kConsumerWarps && lane == 0 && !p.idle_producer;
    const int first_claim = producer ? atomicAdd(&p.ctrl[0], 1) : 0;
    const Plan pl = plan_items(p, sm.off, sm.red);

    // Rows without a cached token (CUDA-graph padding) have no items and get a zero output.
    const int64_t row_vec = int64_t(p.lq) * p.hq * kD / 8;  // uint4 per batch row
    for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
        if (sm.off[b + 1] == sm.off[b]) {
            uint4* o = reinterpret_cast<uint4*>(p.out) + b * row_vec;
            for (int64_t i = tid; i < row_vec; i += kThreads) o[i] = make_uint4(0, 0, 0, 0);
        }
    }

    if (warp == kConsumerWarps) {
        // ------------------------------------------------------------ producer
        if (producer) {
            const uint64_t pol = l2_policy_evict_first();
            const uint32_t q_bytes = uint32_t(p.group) * kD * 2;  // one query token's rows of this kv head
            int stage = 0;
            uint32_t phase = 0;
            int64_t fills = 0;
            bool ok = true;
            ItemMeta cur, nxt;
            cur.item = pl.total_items;
            if (first_claim < pl.total_items) fetch_meta(cur, first_claim, p, sm.off, pl.total_full, pl.chunk, pl.cap);
            while (ok && cur.item < pl.total_items) {
                const int ctx = min(cur.ctx, pl.cap);
                const int nt = (ctx + kTile - 1) / kTile;
                const int t0 = cur.t0;
                const int t1 = int(min(int64_t(nt), t0 + pl.chunk));
                const int32_t* bt = p.block_tables + int64_t(cur.b) * p.bt_stride;
                const int t_claim = max(t0, t1 - kClaimAhead);
                nxt.item = pl.total_items;
                for (int t = t0; t < t1; ++t) {
                    if (!mbar_wait(&sm.empty[stage], phase ^ 1, p.wait_ns)) {
                        atomicOr(&p.ctrl[2], DEV_ERR_WAIT_EMPTY);
                        ok = false;
                        break;
                    }
                    const bool first = t == t0;
                    const int pos = t * kTile;
                    const int lb = pos / p.block_size;
                    int blk;
                    const int j = lb - cur.page0;
                    if (j < kPrefetchPages) {
                        blk = cur.blk[0];
#pragma unroll
                        for (int u = 1; u < kPrefetchPages; ++u)
                            if (j == u) blk = cur.blk[u];
                    } else {
                        blk = bt[lb];
                    }
                    const bool page = blk >= 0 && blk < p.num_blocks;
                    Header& hd = sm.hdr[stage];
                    hd.item = cur.item;
                    hd.b = cur.b;
                    hd.h = cur.h;
                    hd.tile = t;
                    hd.flags = (first ? kFirst : 0) | (t == t1 - 1 ? kLast : 0) | (page ? 0 : kNoPage);
                    hd.ctx = ctx;
                    hd.nchunks = cur.nchunks;
                    hd.slot0 = cur.slot0;
                    mbar_arrive_expect_tx(&sm.full[stage], (page ? uint32_t(kStage) : 0u) + (first ? q_bytes * p.lq : 0u));
                    uint8_t* st = sm.stages[stage];
                    if (page) {
                        const int64_t o = ((int64_t(blk) * p.hkv + cur.h) * p.block_size + (pos - lb * p.block_size)) * kRecord;
                        bulk_load_hint(st, qp.k + o, kKvBytes, &sm.full[stage], pol);
                        bulk_load_hint(st + kKvBytes, qp.v + o, kKvBytes, &sm.full[stage], pol);
                    }
                    if (first) {
                        const uint16_t* qsrc = p.q + int64_t(cur.b) * p.lq * p.q_stride + int64_t(cur.h) * p.group * kD;
                        for (int jq = 0; jq < p.lq; ++jq)
                            bulk_load(sm.qbuf[stage] + jq * q_bytes, qsrc + int64_t(jq) * p.q_stride, q_bytes,
                                      &sm.full[stage]);
                    }
                    ++fills;
                    if (++stage == NS) { stage = 0; phase ^= 1; }
                    if (t == t_claim) {  // the claim's dependent loads overlap the tiles in flight
                        const int claim = atomicAdd(&p.ctrl[0], 1);
                        if (claim < pl.total_items) fetch_meta(nxt, claim, p, sm.off, pl.total_full, pl.chunk, pl.cap);
                    }
                }
                cur = nxt;
            }
            if (ok) {
                if (mbar_wait(&sm.empty[stage], phase ^ 1, p.wait_ns)) {
                    sm.hdr[stage].item = -1;  // sentinel: no more tiles
                    mbar_arrive(&sm.full[stage]);
                } else {
                    atomicOr(&p.ctrl[2], DEV_ERR_WAIT_EMPTY);
                    ok = false;
                }
            }
            if (!ok) {
                // Error path: wait (bounded) for every copy still in flight before the CTA's
                // shared memory is released.
                for (int s = 0; s < NS; ++s) {
                    if (fills <= s) break;
                    const int64_t last = s + ((fills - 1 - s) / NS) * NS;
                    if (!mbar_wait(&sm.full[s], uint32_t((last / NS) & 1), p.wait_ns))
                        atomicOr(&p.ctrl[2], DEV_ERR_WAIT_DRAIN);
                }
            }
        }
        __syncwarp();
    } else {
        // ------------------------------------------------------------ consumers
        const int g = lane >> 2, c = lane & 3;
        // Byte offset in a stage of the 16-byte row this lane hands to ldmatrix: token (lane & 7) of
        // the warp's 16, group lane >> 3; and of the parameters of token g.
        const uint32_t frag_off = uint32_t(warp * 16 + (lane & 7)) * kRecord + (lane >> 3) * 16;
        const uint32_t par_off = uint32_t(warp * 16 + g) * kRecord + q4::kParams;
        int stage = 0;
        uint32_t phase = 0, cphase = 0;
        // Query rows 8 nt + 2 c + j: reference r (log2), sum l, score factor f, group sums of q, limits.
        float r_ref[NT][2], l_run[NT][2], fac[NT][2], qsum[kGroups][NT][2];
        int lim[NT][2];
        int lim_min = 0;
        float o[kGroups][2][NT][4];   // O^T fragments: 16 dims x 8 rows, in units of 2^-24 and 2^-20
        float om[kGroups][NT][2];     // sum_t p m of this lane's tokens
        uint32_t qf[kGroups][2][NT][2];
        int ev = kExpMin;             // E
        float s_lim = 0.f;
        while (true) {
            // Exit decisions are warp-uniform (the lanes' waits can disagree at the limit).
            if (!__all_sync(0xffffffffu, mbar_wait(&sm.full[stage], phase, p.wait_ns))) {
                atomicOr(&p.ctrl[2], DEV_ERR_WAIT_FULL);
                *reinterpret_cast<volatile int32_t*>(&sm.err) = 1;
                break;
            }
            // A sibling consumer warp that gave up will not reach the consumer barrier below.
            if (__any_sync(0xffffffffu, *reinterpret_cast<volatile int32_t*>(&sm.err) != 0)) break;
            const Header hd = sm.hdr[stage];
            if (hd.item < 0) break;
            if (hd.flags & kFirst) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const int row = 8 * nt + g;
                    float x[kGroups][8];
                    float mx = 0.f;
#pragma unroll
                    for (int j = 0; j < kGroups; ++j) {
                        uint4 w = make_uint4(0, 0, 0, 0);
                        if (row < p.rows)
                            w = *reinterpret_cast<const uint4*>(sm.qbuf[stage] + row * kD * 2 + (32 * j + 8 * c) * 2);
                        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            x[j][2 * i] = lo_f<BF16>(u[i]);
                            x[j][2 * i + 1] = hi_f<BF16>(u[i]);
                            mx = fmaxf(mx, fmaxf(fabsf(x[j][2 * i]), fabsf(x[j][2 * i + 1])));
                        }
                    }
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                    // The row times 2^-eq has its largest element in [2^13, 2^14).
                    const int eq = mx > 0.f ? min(max((__float_as_int(mx) >> 23) - 127 - 13, kExpMin), kExpMax) : 0;
                    const float sc = exp2_int(-eq);
                    float sum[kGroups];
#pragma unroll
                    for (int j = 0; j < kGroups; ++j) {
                        sum[j] = 0.f;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            x[j][i] *= sc;
                            sum[j] += x[j][i];
                        }
                        sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 1);
                        sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 2);
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            qf[j][i][nt][0] = pack2<false>(x[j][4 * i], x[j][4 * i + 1]);
                            qf[j][i][nt][1] = pack2<false>(x[j][4 * i + 2] * 0.0625f, x[j][4 * i + 3] * 0.0625f);
                        }
                    }
                    const float f = p.scale_log2 * exp2_int(eq + 24);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int src = (2 * c + e) * 4;  // a lane that holds query row 8 nt + 2 c + e
                        fac[nt][e] = __shfl_sync(0xffffffffu, f, src);
#pragma unroll
                        for (int j = 0; j < kGroups; ++j)
                            qsum[j][nt][e] = __shfl_sync(0xffffffffu, sum[j], src) * 5.9604644775390625e-8f;  // 2^-24
                        const int rw = 8 * nt + 2 * c + e;
                        // Padding rows (past p.rows) see the whole context: only rows that exist mask.
                        lim[nt][e] = rw < p.rows ? hd.ctx - p.lq + rw / p.group : hd.ctx - 1;
                        r_ref[nt][e] = kNone;
                        l_run[nt][e] = 0.f;
                    }
                }
                lim_min = hd.ctx - p.lq;  // row 0's limit, the smallest
                ev = kExpMin;
                s_lim = 0.f;
#pragma unroll
                for (int j = 0; j < kGroups; ++j)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        om[j][nt][0] = om[j][nt][1] = 0.f;
#pragma unroll
                        for (int t = 0; t < 2; ++t)
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[j][t][nt][e] = 0.f;
                    }
            }
            const int tok_base = hd.tile * kTile + warp * 16;
            uint8_t* st = sm.stages[stage];
            bool wrote = false;
            if (tok_base < hd.ctx) {
                // Records past the context may hold anything (a NaN scale times a probability of 0 is
                // NaN), a page outside the cache was not loaded: both read as zeros.
                const int first = (hd.flags & kNoPage) ? 0 : hd.ctx - tok_base;
                if (first < 16) {
                    for (int i = lane; i < (16 - first) * (kRecord / 16); i += 32) {
                        const int at = (warp * 16 + first) * kRecord + i * 16;
                        *reinterpret_cast<uint4*>(st + at) = make_uint4(0, 0, 0, 0);
                        *reinterpret_cast<uint4*>(st + kKvBytes + at) = make_uint4(0, 0, 0, 0);
                    }
                    wrote = true;
                    __syncwarp();
                }
                constexpr uint32_t kLo = 0x000f000fu, kHi = 0x00f000f0u;
                // ---- S^T = K Q^T ----
                uint32_t ka[kGroups], kb[kGroups];  // word c of tokens g and g + 8
                ldsm_x4(ka[0], ka[1], ka[2], ka[3], smem_u32(st) + frag_off);
                ldsm_x4(kb[0], kb[1], kb[2], kb[3], smem_u32(st) + frag_off + 8 * kRecord);
                const uint4 pka4 = *reinterpret_cast<const uint4*>(st + par_off);
                const uint4 pkb4 = *reinterpret_cast<const uint4*>(st + par_off + 8 * kRecord);
                const uint4 pva4 = *reinterpret_cast<const uint4*>(st + kKvBytes + par_off);
                const uint4 pvb4 = *reinterpret_cast<const uint4*>(st + kKvBytes + par_off + 8 * kRecord);
                const uint32_t pka[4] = {pka4.x, pka4.y, pka4.z, pka4.w}, pkb[4] = {pkb4.x, pkb4.y, pkb4.z, pkb4.w};
                float x[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) x[nt][0] = x[nt][1] = x[nt][2] = x[nt][3] = 0.f;
#pragma unroll
                for (int j = 0; j < kGroups; ++j) {
                    const uint32_t a0[4] = {ka[j] & kLo, kb[j] & kLo, ka[j] & kHi, kb[j] & kHi};
                    const uint32_t wa = ka[j] >> 8, wb = kb[j] >> 8;
                    const uint32_t a1[4] = {wa & kLo, wb & kLo, wa & kHi, wb & kHi};
                    const float sa = lo_f<BF16>(pka[j]), ma = hi_f<BF16>(pka[j]);
                    const float sb = lo_f<BF16>(pkb[j]), mb = hi_f<BF16>(pkb[j]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float acc[4] = {0.f, 0.f, 0.f, 0.f};
                        mma_16816<false>(acc, a0, qf[j][0][nt][0], qf[j][0][nt][1]);
                        mma_16816<false>(acc, a1, qf[j][1][nt][0], qf[j][1][nt][1]);
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            x[nt][e] = fmaf(sa, acc[e], fmaf(ma, qsum[j][nt][e], x[nt][e]));
                            x[nt][2 + e] = fmaf(sb, acc[2 + e], fmaf(mb, qsum[j][nt][e], x[nt][2 + e]));
                        }
                    }
                }
                // ---- log2 probabilities, masks, running references ----
                const bool edge = tok_base + 15 > lim_min;  // the tile reaches past some row's last visible token
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[nt][e] *= fac[nt][e & 1];
                if (edge) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (tok_base + g + (e >> 1) * 8 > lim[nt][e & 1]) x[nt][e] = -INFINITY;
                }
                float sva[4], svb[4], mva[4], mvb[4];
                {
                    const uint32_t pa[4] = {pva4.x, pva4.y, pva4.z, pva4.w}, pb[4] = {pvb4.x, pvb4.y, pvb4.z, pvb4.w};
#pragma unroll
                    for (int j = 0; j < kGroups; ++j) {
                        sva[j] = lo_f<BF16>(pa[j]);
                        mva[j] = hi_f<BF16>(pa[j]);
                        svb[j] = lo_f<BF16>(pb[j]);
                        mvb[j] = hi_f<BF16>(pb[j]);
                    }
                }
                const float s_max = fmaxf(max3f(max3f(sva[0], sva[1], sva[2]), sva[3], svb[0]), max3f(svb[1], svb[2], svb[3]));
                float y_max = -INFINITY;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) y_max = fmaxf(y_max, x[nt][e] - r_ref[nt][e & 1]);
                if (__any_sync(0xffffffffu, y_max > kLazyMax - float(ev) || s_max > s_lim)) {
                    // Rare: raise E to the value scales of this tile, the rows' maxima to its scores.
                    float sm_all = s_max;
#pragma unroll
                    for (int sh = 1; sh <= 16; sh <<= 1) sm_all = fmaxf(sm_all, __shfl_xor_sync(0xffffffffu, sm_all, sh));
                    int raise = 0;
                    if (sm_all > s_lim) {
                        const int en = min(max((__float_as_int(sm_all) >> 23) - 127 - 2, ev), kExpMax);
                        raise = en - ev;
                        ev = en;
                        s_lim = en == kExpMax ? INFINITY : exp2_int(en + 7);
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float tm = fmaxf(x[nt][e], x[nt][2 + e]);
#pragma unroll
                            for (int sh = 4; sh <= 16; sh <<= 1) tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, sh));
                            const float ro = r_ref[nt][e];
                            const float rn = fmaxf(ro == kNone ? kNone : ro + float(raise), tm == -INFINITY ? kNone : tm + float(ev));
                            const float alpha = ro == kNone ? 0.f : fast_exp2(ro - rn);
                            r_ref[nt][e] = rn;
                            l_run[nt][e] *= alpha;
#pragma unroll
                            for (int j = 0; j < kGroups; ++j) {
                                om[j][nt][e] *= alpha;
#pragma unroll
                                for (int t = 0; t < 2; ++t) {
                                    o[j][t][nt][e] *= alpha;
                                    o[j][t][nt][2 + e] *= alpha;
                                }
                            }
                        }
                }
                float pr[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) pr[nt][e] = fast_exp2(x[nt][e] - r_ref[nt][e & 1]);
                    l_run[nt][0] += pr[nt][0] + pr[nt][2];
                    l_run[nt][1] += pr[nt][1] + pr[nt][3];
                }
                if (edge) {
                    // A stored non-finite value (s = m = NaN) counts for the rows that see its token only.
#pragma unroll
                    for (int j = 0; j < kGroups; ++j) {
                        const bool bad_a = !(fabsf(sva[j]) <= FLT_MAX && fabsf(mva[j]) <= FLT_MAX);
                        const bool bad_b = !(fabsf(svb[j]) <= FLT_MAX && fabsf(mvb[j]) <= FLT_MAX);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 2; ++e)
                                if ((bad_a && pr[nt][e] != 0.f) || (bad_b && pr[nt][2 + e] != 0.f))
                                    om[j][nt][e] = __int_as_float(0x7fffffff);
                        if (bad_a) sva[j] = mva[j] = 0.f;
                        if (bad_b) svb[j] = mvb[j] = 0.f;
                    }
                }
                // ---- O^T += V^T (P s)^T, and the minima's part ----
                uint32_t va[kGroups], vb[kGroups];  // half-word g of tokens 2 c, 2 c + 1 (va) and 2 c + 8, 2 c + 9 (vb)
                ldsm_x4_t(va[0], va[1], va[2], va[3], smem_u32(st) + kKvBytes + frag_off);
                ldsm_x4_t(vb[0], vb[1], vb[2], vb[3], smem_u32(st) + kKvBytes + frag_off + 8 * kRecord);
#pragma unroll
                for (int j = 0; j < kGroups; ++j) {
                    uint32_t b[NT][2];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        b[nt][0] = movmatrix_t(pack2<false>(pr[nt][0] * sva[j], pr[nt][1] * sva[j]));
                        b[nt][1] = movmatrix_t(pack2<false>(pr[nt][2] * svb[j], pr[nt][3] * svb[j]));
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            om[j][nt][e] = fmaf(pr[nt][e], mva[j], fmaf(pr[nt][2 + e], mvb[j], om[j][nt][e]));
                    }
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const uint32_t wa = va[j] >> (8 * t), wb = vb[j] >> (8 * t);
                        const uint32_t a[4] = {wa & kLo, wa & kHi, wb & kLo, wb & kHi};
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma_16816<false>(o[j][t][nt], a, b[nt][0], b[nt][1]);
                    }
                }
            }
            if (wrote) fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.empty[stage]);
            if (++stage == NS) { stage = 0; phase ^= 1; }

            if (hd.flags & kLast) {
                // ---- combine the eight warps' states of this item ----
                // Sums over the lanes that hold the same rows (all g), then O = 2^24 o + sum p m.
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
#pragma unroll
                        for (int sh = 4; sh <= 16; sh <<= 1)
                            l_run[nt][e] += __shfl_xor_sync(0xffffffffu, l_run[nt][e], sh);
#pragma unroll
                        for (int j = 0; j < kGroups; ++j) {
#pragma unroll
                            for (int sh = 4; sh <= 16; sh <<= 1)
                                om[j][nt][e] += __shfl_xor_sync(0xffffffffu, om[j][nt][e], sh);
#pragma unroll
                            for (int t = 0; t < 2; ++t) {
                                o[j][t][nt][e] = fmaf(o[j][t][nt][e], 16777216.f, om[j][nt][e]);
                                o[j][t][nt][2 + e] = fmaf(o[j][t][nt][2 + e], 1048576.f, om[j][nt][e]);
                            }
                        }
                    }
                constexpr int kHalf = kConsumerWarps / 2;
                // Dimension of o[j][t][.][e] for e < 2; e >= 2 is the next nibble, two dimensions on.
                const int d0 = 8 * (g >> 1) + (g & 1);
                // 8 -> 4: warps 4-7 hand their state to warps 0-3, which merge it in registers.
                if (warp >= kHalf) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int r = 8 * nt + 2 * c + e;
                            if (g == 0) {
                                sm.cm[warp][r] = r_ref[nt][e];
                                sm.cl[warp][r] = l_run[nt][e];
                            }
#pragma unroll
                            for (int j = 0; j < kGroups; ++j)
#pragma unroll
                                for (int t = 0; t < 2; ++t) {
                                    float* cp = &sm.co[warp - kHalf][r][32 * j + 4 * t + d0];
                                    cp[0] = o[j][t][nt][e];
                                    cp[2] = o[j][t][nt][2 + e];
                                }
                        }
                }
                if (!consumer_sync(&sm.cbar, cphase, p.wait_ns)) {
                    atomicOr(&p.ctrl[2], DEV_ERR_WAIT_PEER);
                    *reinterpret_cast<volatile int32_t*>(&sm.err) = 1;
                    break;
                }
                if (warp < kHalf) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int r = 8 * nt + 2 * c + e;
                            const float mb = sm.cm[warp + kHalf][r], lb = sm.cl[warp + kHalf][r];
                            const float M = fmaxf(r_ref[nt][e], mb);
                            const float wa = fast_exp2(r_ref[nt][e] - M), wb = fast_exp2(mb - M);
#pragma unroll
                            for (int j = 0; j < kGroups; ++j)
#pragma unroll
                                for (int t = 0; t < 2; ++t) {
                                    float* cp = &sm.co[warp][r][32 * j + 4 * t + d0];
                                    cp[0] = o[j][t][nt][e] * wa + cp[0] * wb;
                                    cp[2] = o[j][t][nt][2 + e] * wa + cp[2] * wb;
                                }
                            if (g == 0) {
                                sm.cm[warp][r] = M;
                                sm.cl[warp][r] = l_run[nt][e] * wa + lb * wb;
                            }
                        }
                }
                if (!consumer_sync(&sm.cbar, cphase, p.wait_ns)) {
                    atomicOr(&p.ctrl[2], DEV_ERR_WAIT_PEER);
                    *reinterpret_cast<volatile int32_t*>(&sm.err) = 1;
                    break;
                }
                // 4 -> 1 over shared memory, one output element per thread and round.
                const bool single = hd.nchunks == 1;
                const int nel = p.rows * kD;
                const int cslot = hd.item / p.hkv;  // this chunk's partial slot (before x Hkv + h)
                for (int idx = tid; idx < nel; idx += kConsumers) {
                    const int r = idx >> 7, d = idx & (kD - 1);
                    float M = sm.cm[0][r];
#pragma unroll
                    for (int w = 1; w < kHalf; ++w) M = fmaxf(M, sm.cm[w][r]);
                    float den = 0.f, acc = 0.f;
#pragma unroll
                    for (int w = 0; w < kHalf; ++w) {
                        const float sc = fast_exp2(sm.cm[w][r] - M);
                        den = fmaf(sm.cl[w][r], sc, den);
                        acc = fmaf(sm.co[w][r][d], sc, acc);
                    }
                    const float val = den == 0.f ? 0.f : acc / den;  // 0: the row sees no token of this item
                    if (single) {
                        const int j = r / p.group, gq = r - j * p.group;
                        p.out[((int64_t(hd.b) * p.lq + j) * p.hq + hd.h * p.group + gq) * kD + d] = to_bits16<BF16>(val);
                    } else {
                        const int64_t it = int64_t(cslot) * p.hkv + hd.h;
                        p.part_o[(it * p.rows + r) * kD + d] = val;
                        // A NaN sum is handed on as an infinite weight: the merge's maximum skips NaN.
                        if (d == 0)
                            p.part_lse[it * p.rows + r] =
                                den == 0.f ? -INFINITY : (den <= FLT_MAX ? M + fast_log2(den) : INFINITY);
                    }
                }
                if (!single) {
                    // Publish this chunk (one release fence per CTA, cumulative over the barrier), then
                    // count it; the last chunk's CTA merges.
                    if (!consumer_sync(&sm.cbar, cphase, p.wait_ns)) {
                        atomicOr(&p.ctrl[2], DEV_ERR_WAIT_PEER);
                        *reinterpret_cast<volatile int32_t*>(&sm.err) = 1;
                        break;
                    }
                    if (tid == 0) {
                        __threadfence();
                        const int prev = atomicAdd(&p.counters[hd.b * p.hkv + hd.h], 1);
                        const bool last = prev == hd.nchunks - 1;
                        if (last) __threadfence();
                        sm.flag = last;
                    }
                    if (!consumer_sync(&sm.cbar, cphase, p.wait_ns)) {
                        atomicOr(&p.ctrl[2], DEV_ERR_WAIT_PEER);
                        *reinterpret_cast<volatile int32_t*>(&sm.err) = 1;
                        break;
                    }
                    if (sm.flag) {
                        merge_chunks<BF16>(p, hd, pl, tid);
                        if (tid == 0) p.counters[hd.b * p.hkv + hd.h] = 0;
                    }
                }
                if (!consumer_sync(&sm.cbar, cphase, p.wait_ns)) {
                    atomicOr(&p.ctrl[2], DEV_ERR_WAIT_PEER);
                    *reinterpret_cast<volatile int32_t*>(&sm.err) = 1;
                    break;
                }
            }
        }
    }

    __syncthreads();
    if (tid == 0) {
        __threadfence();
        const int done = atomicAdd(&p.ctrl[1], 1);
        if (done == int(gridDim.x) - 1) {
            // Every CTA has stopped claiming items: re-arm the scheduler.
            atomicExch(&p.ctrl[0], 0);
            atomicExch(&p.ctrl[1], 0);
        }
    }
}

template <bool BF16, int NT>
void launch(const Q4Params& prm, cudaStream_t s) {
    const void* fn = (const void*)paged_attention_q4_kernel<BF16, NT>;
    ensure_smem_attr(fn, int(sizeof(Smem<NT>)));
    paged_attention_q4_kernel<BF16, NT>
        <<<device_sm_count() * Cfg<NT>::kCtas, kThreads, sizeof(Smem<NT>), s>>>(prm);
}

}  // namespace
}  // namespace pa
}  // namespace b200

extern "C" int32_t b200_paged_attention_q4(void* out, const void* q, int64_t q_stride_token, const void* k_cache,
                                           const void* v_cache, int32_t num_blocks, int32_t block_size,
                                           const int32_t* block_tables, int64_t block_table_stride,
                                           int32_t block_table_width, const int32_t* context_lens, int32_t batch, int32_t query_len,
                                           int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                           float softmax_scale, int32_t dtype, void* workspace, size_t workspace_bytes,
                                           void* stream) {
    using namespace b200;
    using namespace b200::pa;
    clear_error();
    B200_REQUIRE(batch >= 0, "paged_attention_q4: batch %d < 0", batch);
    if (batch == 0) return B200_OK;
    B200_REQUIRE(out && q && k_cache && v_cache && block_tables && context_lens, "paged_attention_q4: null pointer");
    B200_REQUIRE(num_heads > 0 && num_kv_heads > 0 && num_heads % num_kv_heads == 0,
                 "paged_attention_q4: num_heads %d not a multiple of num_kv_heads %d", num_heads, num_kv_heads);
    B200_REQUIRE(query_len >= 1, "paged_attention_q4: query_len %d < 1", query_len);
    B200_REQUIRE(softmax_scale > 0.f && softmax_scale <= FLT_MAX,
                 "paged_attention_q4: softmax_scale %g not positive and finite", double(softmax_scale));
    const int group = num_heads / num_kv_heads;
    const int64_t rows = int64_t(query_len) * group;
    if (head_dim != kD) return fail(B200_ERR_UNSUPPORTED, "paged_attention_q4: head_dim %d (only 128)", head_dim);
    if (rows > 16)
        return fail(B200_ERR_UNSUPPORTED, "paged_attention_q4: query_len * Hq/Hkv = %lld exceeds 16", (long long)rows);
    if (dtype != B200_BF16 && dtype != B200_F16)
        return fail(B200_ERR_UNSUPPORTED, "paged_attention_q4: dtype %d (bf16 or fp16 only)", dtype);
    if (batch > kMaxBatch) return fail(B200_ERR_UNSUPPORTED, "paged_attention_q4: batch %d > %d", batch, kMaxBatch);
    B200_REQUIRE(block_size > 0 && block_size % kTile == 0, "paged_attention_q4: block_size %d not a multiple of %d",
                 block_size, kTile);
    B200_REQUIRE(num_blocks > 0 && int64_t(num_blocks) * block_size < (int64_t(1) << 31),
                 "paged_attention_q4: num_blocks %d out of range", num_blocks);
    B200_REQUIRE(block_table_width > 0 && int64_t(block_table_width) * block_size < (int64_t(1) << 31) &&
                     block_table_stride >= 0 && block_table_stride <= INT32_MAX,
                 "paged_attention_q4: block table of %d entries, stride %lld out of range", block_table_width,
                 (long long)block_table_stride);
    auto al16 = [](const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15) == 0; };
    B200_REQUIRE(q_stride_token >= int64_t(num_heads) * head_dim && q_stride_token % 8 == 0 && al16(q) && al16(out) &&
                     al16(k_cache) && al16(v_cache),
                 "paged_attention_q4: q, out and the caches must be 16-byte aligned, q token stride (%lld) a multiple of 8 "
                 "and at least Hq*D",
                 (long long)q_stride_token);
    if (int64_t(batch) * num_kv_heads > kCounterSlots)
        return fail(B200_ERR_UNSUPPORTED, "paged_attention_q4: batch * num_kv_heads > %d", kCounterSlots);
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) || workspace_bytes < kFixedBytes)
        return fail(B200_ERR_WORKSPACE, "paged_attention_q4: workspace missing, unaligned or smaller than %zu bytes",
                    kFixedBytes);
    const int64_t max_items = int64_t(workspace_bytes - kFixedBytes) / (rows * (kD + 1) * 4);
    if (max_items < int64_t(batch) * num_kv_heads)
        return fail(B200_ERR_WORKSPACE, "paged_attention_q4: workspace holds %lld items, batch * Hkv = %lld",
                    (long long)max_items, (long long)batch * num_kv_heads);

    Q4Params prm;
    prm.k = static_cast<const uint8_t*>(k_cache);
    prm.v = static_cast<const uint8_t*>(v_cache);
    Params& b = prm.base;
    b.q = static_cast<const uint16_t*>(q);
    b.q_stride = q_stride_token;
    b.out = static_cast<uint16_t*>(out);
    b.block_tables = block_tables;
    b.bt_stride = int32_t(block_table_stride);
    b.bt_width = block_table_width;
    b.context_lens = context_lens;
    b.batch = batch;
    b.lq = query_len;
    b.hq = num_heads;
    b.hkv = num_kv_heads;
    b.group = group;
    b.rows = int32_t(rows);
    b.block_size = block_size;
    b.num_blocks = num_blocks;
    b.scale_log2 = softmax_scale * 1.4426950408889634f;
    char* ws = static_cast<char*>(workspace);
    b.ctrl = reinterpret_cast<int32_t*>(ws);
    b.counters = reinterpret_cast<int32_t*>(ws + kCtrlWords * 4);
    b.part_o = reinterpret_cast<float*>(ws + kFixedBytes);
    b.part_lse = b.part_o + max_items * rows * kD;
    b.max_items = int32_t(max_items > INT32_MAX / 2 ? INT32_MAX / 2 : max_items);
    apply_test_hook(b);

    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool wide = rows > 8;
    if (dtype == B200_BF16) {
        if (wide) launch<true, 2>(prm, s);
        else launch<true, 1>(prm, s);
    } else {
        if (wide) launch<false, 2>(prm, s);
        else launch<false, 1>(prm, s);
    }
    B200_CUDA_TRY(cudaGetLastError());
    return B200_OK;
}
