// Paged multi-query attention for decode and speculative verification over a 4-bit KV cache:
// the call of nanovllm/layers/attention.py:71-74 on records of kv_q4.cuh.
//
// Mathematics.  A cached value is s n + m with n the 4-bit code and one (s, m) per group of 32
// head dimensions, so per query row and token
//     q . k = sum_g s_g (q_g . n_g) + sum_g m_g sum(q_g),    o_g = sum_t (p_t s_tg) n_tg + sum_t p_t m_tg.
// The codes themselves are the matrix operands: a nibble in the low bits of an fp16 lane is the
// subnormal n * 2^-24 (16 n * 2^-24 one nibble up), exactly, so that a mask turns a word of
// codes into operands of mma.sync.m16n8k16 and nothing is converted.  The powers of two are
// undone in fp32; the queries that meet a second nibble carry a factor 1/16.  (A product of 16 terms cuts
// each at 2^-25 of the largest exponent sum of its operands, in which a subnormal counts as 2^-14: what is
// lost is below 2^-15 of code 1 times the largest other operand, per term.)
//   * Tokens are the M of both products' operands: S^T = K Q^T and O^T = V^T (P s)^T, query rows
//     their N of 8.  ldmatrix hands lane (g, c) word c of token g's four groups, the transposed form
//     half-word g of tokens 2 c and 2 c + 1: one nibble per dimension (token) in either half of a
//     register both times.  For the values the second operand row is the byte n + 16 n' as it is:
//     n' comes out by subtraction at the end, which saves a mask.  P^T turns into a B operand by
//     movmatrix.
//   * The words (s, m) of a token are operands too: against the rows (0, sum(q_g)), in two fp16 or
//     three bf16 parts (22 or 24 bits), they give the minima's part of the score; taken to fp16
//     (times a power of two) and transposed, against P^T, sum_t p m, and with a row of ones beside
//     them the softmax sum.
//   * The key scales multiply the products in fp32.  The value scales multiply P^T in fp16: the
//     lanes of row 2 g of the transposed words hold them, one shuffle hands them round.
// Roundings: p to fp16 (2^-11), the same rounded p in the products and in the sum, so that the
// result is a mean under weights off by as much; p s to fp16 (2^-11).  fp16 models, whose outputs
// would show both, carry the rest of p and of p s in a second product (0.00023 from 64 bits
// relative, 0.00034 without; the output's own rounding is 0.0002).  Sums and maxima are fp32, but
// for what a matrix product cuts (above).
//
// Ranges.  p = 2^(x - r) with r lazily raised to 2^8 below the running maximum, so p <= 2^kLazyMax.  The
// value parameters enter as 2^-E of themselves, one E per group, which follows the group's largest
// max(16 s, |m|) that the warp has met (below 2^4 in these units when E is set, raised beyond 2^7): a
// group keeps its precision beside far larger ones.  Queries are scaled by a power of two per row
// (largest element in [8, 16)), exactly but for elements below 2^-18 of it.
//
// Work split.  The tiles of 128 tokens of all (sequence, kv head) pairs in a row, sequence by
// sequence, are cut into equal runs (a pair counts kPairCost tiles more for its combine), one per
// CTA, all CTAs resident: no claims, a sequence is split only where a run ends, and a long one over
// as many CTAs as its share of the work.  Every CTA plans its run from context_lens (no host sync:
// the call can be captured).  A CTA leaves at most two partial results, its first and its last; the
// warp that finishes the last chunk of a split pair (one counter per consumer warp) merges its
// share of the outputs, many chunks in groups first.
//
// CTA.  Four consumer warps and a producer warp; three CTAs per SM up to 8 query rows (15 warps
// leave 128 registers a thread), two for up to 16 (168).  A stage is 128 records of keys and 128 of
// values, two contiguous 10 KiB bulk copies into a ring of two, guarded by full / empty mbarriers;
// each consumer warp takes 32 of a tile's tokens, in two sub-tiles of 16.  The warps keep their own
// softmax states and combine them through shared memory at the end of an item.  Every wait is
// bounded (kWaitLimitNs, or the test limit).
//
// What bounds it (512 sequences, 1.17 M tokens, 8 kv heads of 4 rows: 1.50 GB, 228 us at the measured
// copy rate): 267 us, 158 M warp instructions, the vector pipes; held for a second it reaches the
// board's power cap, 1.69 GHz and 310 to 313 us.  A record costs its share of 271 instructions per
// 16 tokens, 72 of them masks.  16 consumer warps per SM (104 registers each, taken from their
// producers) issue more often, spill, and gain nothing; they would cost the short calls 2 us.
#include <atomic>
#include <cfloat>
#include <climits>
#include <type_traits>

#include "kv_q4.cuh"

namespace b200 {
namespace pq4 {
namespace {

using q4::hi_f;
using q4::kD;
using q4::kGroups;
using q4::kRecord;
using q4::lo_f;

constexpr int kTile = 128;  // tokens per stage
constexpr int kWarps = 4;   // consumer warps
constexpr int kWarpTokens = kTile / kWarps;
constexpr int kConsumers = kWarps * 32;
constexpr int kThreads = kConsumers + 32;
constexpr int kStages = 2;
// Items whose query rows fit: rows are taken with an item's first tile, so a buffer is free again when
// the stage that is filled next is.
constexpr int kQBufs = kStages;
constexpr int kKvBytes = kTile * kRecord;  // keys (or values) of one stage
constexpr int kStageBytes = 2 * kKvBytes;
constexpr int kMaxBatch = 2048;
// What a (sequence, kv head) pair costs beside its tiles, in tiles (decode of 512 sequences / verify of
// 128: 272 / 129 us with 2, 275 / 138 with 1, 277 / 130 with 3, 282 / 132 with 4).
constexpr int kPairCost = 2;
constexpr float kCodeUnit = 1.f / 16777216.f;  // 2^-24, the value of code 1 as an fp16 operand
// A row's reference is set kTop (log2) below its maximum and raised once a score exceeds it by kLazyMax: the
// largest p lies in [2^8, 2^12].  fp16 ends at 2^-25, so a token keeps a weight down to 2^-33 of the largest one's:
// a long tail behind one token of a far larger score is not lost.  (p s stays below 2^15: kReach.)
constexpr float kTop = 8.f;
constexpr float kLazyMax = 12.f;
// What value parameters (16 s, |m|) times 2^-E may reach before E is raised, to where they lie in [2^kUnitBits, 2 * that).
constexpr float kReach = 128.f;
constexpr int kUnitBits = 3;
constexpr float kNone = -1e30f;  // reference of a row that has met no token
constexpr int kExpMax = 60;      // bound of |E| and of the query rows' exponents

struct Params {
    const uint16_t* q;
    int64_t q_stride;
    uint16_t* out;
    const uint8_t* k;
    const uint8_t* v;
    const int32_t* block_tables;
    int64_t bt_stride;
    int32_t bt_width;
    const int32_t* context_lens;
    int32_t batch, lq, hq, hkv, group, rows, block_size, num_blocks;
    int32_t group_inv;  // ceil(2^16 / group): r / group = (r * group_inv) >> 16 for r < 16
    float scale_log2;
    uint64_t wait_ns;       // limit of every wait (kWaitLimitNs; shorter under the idle-producer test)
    int32_t idle_producer;  // test hook: 1 every producer, 2 + n that of CTA n issues nothing, so a wait runs out
    int32_t* error;
    int32_t* counters;
    float* part_o;    // [2 * CTAs][rows][kD]
    float* part_lse;  // [2 * CTAs][kWarps][rows]
};

// What a tile's warps need.
struct alignas(16) TileHeader {
    int32_t tile, flags, ctx, pad;
};
// What is needed at the end of an item: its pair, the CTA of the pair's first chunk, the number of chunks.
struct alignas(16) Header {
    int32_t b, h, first, nch;
};
enum : int32_t { kFirst = 1, kLast = 2, kNoPage = 4, kQBuf = 8 };

// NT: groups of 8 query rows (2 for 9 to 16 rows).
template <int NT>
struct Cfg {
    // Per SM.  Up to 8 rows take 128 registers a thread, which 15 warps leave; up to 16 take 168.
    static constexpr int kCtas = NT == 1 ? 3 : 2;
    static constexpr int kPassRows = NT == 1 ? 4 : 16;  // rows combined at a time (what shared memory leaves)
};

// All CTAs of the grid are resident.
int grid_ctas(int rows) { return device_sm_count() * (rows > 8 ? Cfg<2>::kCtas : Cfg<1>::kCtas); }

// Workspace: control words ([2] error word), counters of the CTAs' last items (one per consumer
// warp; the larger grid's, so that calls of any number of rows can take turns on one workspace), two
// partial results per CTA and, once per consumer warp, their log-sum-exps.
constexpr size_t kCtrlBytes = 256;
size_t fixed_bytes() { return kCtrlBytes + ((size_t(grid_ctas(1)) * kWarps * 4 + 255) & ~size_t(255)); }
static_assert(Cfg<1>::kCtas >= Cfg<2>::kCtas, "fixed_bytes() is the larger grid's");
size_t workspace_bytes(int rows) {
    const int ctas = grid_ctas(rows);
    return (fixed_bytes() + size_t(2) * ctas * rows * (kD + kWarps) * 4 + 255) & ~size_t(255);
}

constexpr int kRowPad = kD + 1;  // floats: the lanes of a fragment write 32 different banks

template <int NT>
struct Smem {
    alignas(128) uint8_t stages[kStages][kStageBytes];
    uint8_t qbuf[kQBufs][8 * NT * kD * 2];
    float co[kWarps][Cfg<NT>::kPassRows][kRowPad];
    float cm[kWarps][Cfg<NT>::kPassRows];
    float cl[kWarps][Cfg<NT>::kPassRows];
    TileHeader tile[kStages];
    Header item[kStages];          // with an item's last tile
    Header part[kWarps][2];        // the run's partial items, as each warp left them
    uint64_t full[kStages];
    uint64_t empty[kStages];
    uint64_t cbar;
    int32_t off[kConsumers / 2];  // length before each entry of 2 ceil(batch / 128) sequences
    int32_t lens[kMaxBatch];      // context lengths in [0, cap]
    int32_t red[kWarps];
    int32_t err;
};
static_assert(sizeof(Smem<1>) <= 233472 / Cfg<1>::kCtas - 1024 && sizeof(Smem<2>) <= 233472 / Cfg<2>::kCtas - 1024,
              "shared memory over the SM's");

__device__ __forceinline__ void bulk_load_hint(void* dst, const void* src, uint32_t bytes, uint64_t* bar,
                                               uint64_t policy) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(
            smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_u32(bar)), "l"(policy)
        : "memory");
}

// D(16x8, f32) = A(16x16) * B(16x8) + C.  Not volatile, unlike common.cuh's: the compiler may order
// these among the loads and conversions.
template <bool BF16>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF16) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    } else {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}
// The same with C = 0, which takes no registers.
template <bool BF16>
__device__ __forceinline__ void mma_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF16) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
    } else {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
    }
}
// movmatrix_t (common.cuh), not volatile.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ float exp2_int(int e) { return __int_as_float((127 + e) << 23); }  // -126 <= e <= 127

// Two fp16 parts of a pair of floats: hi + lo = x to 22 bits.
__device__ __forceinline__ void split2(float2 x, uint32_t& hi, uint32_t& lo) {
    hi = pack2<false>(x.x, x.y);
    const float2 r = fsub2(x, make_float2(lo_f<false>(hi), hi_f<false>(hi)));
    lo = pack2<false>(r.x, r.y);
}

// A pair of 16-bit floats with its infinities and NaNs replaced by zeros.
template <bool BF16>
__device__ __forceinline__ uint32_t finite2(uint32_t w) {
    constexpr uint32_t kExp = BF16 ? 0x7f80u : 0x7c00u;
    if ((w & kExp) == kExp) w &= 0xffff0000u;
    if (((w >> 16) & kExp) == kExp) w &= 0xffffu;
    return w;
}

__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint32_t fma_f16x2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}

// The larger magnitudes of two pairs (their signs are no matter); a NaN beside a number is dropped.
template <bool BF16>
__device__ __forceinline__ uint32_t max_abs(uint32_t a, uint32_t b) {
    uint32_t d;
    if constexpr (BF16) asm("max.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    else asm("max.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

// Two 8x8 matrices of 16-bit elements, as they lie or transposed; lanes 0-15 hand their rows.
__device__ __forceinline__ void ldsm_x2(uint32_t& a, uint32_t& b, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];" : "=r"(a), "=r"(b) : "r"(addr));
}
__device__ __forceinline__ void ldsm_x2_t(uint32_t& a, uint32_t& b, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];" : "=r"(a), "=r"(b) : "r"(addr));
}

// Barrier of the consumer threads, bounded.  False, for the whole warp alike, when a lane's wait ran out.
__device__ __forceinline__ bool consumer_wait(uint64_t* bar, uint32_t& phase, uint64_t limit_ns) {
    const bool ok = mbar_wait_spin(bar, phase, limit_ns);
    phase ^= 1;
    return __all_sync(0xffffffffu, ok);
}

__device__ __forceinline__ int tiles_of(int ctx) { return (ctx + kTile - 1) / kTile; }

__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}

// Counts one arrival: what the warp wrote before is visible to whoever counts after it, and the other way round.
__device__ __forceinline__ int atomic_inc_acq_rel(int32_t* at) {
    int old;
    asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(old) : "l"(at) : "memory");
    return old;
}

// Length of a pair of nt tiles on the line that is cut into runs: its tiles, then kPairCost.
__device__ __forceinline__ int span_of(int nt) { return nt > 0 ? nt + kPairCost : 0; }

// Offset of output row r (query r / group, head r % group of kv head h) of sequence b.
__device__ __forceinline__ int64_t out_row(const Params& p, int b, int h, int r) {
    const int j = (r * p.group_inv) >> 16;
    return ((int64_t(b) * p.lq + j) * p.hq + h * p.group + (r - j * p.group)) * kD;
}

// log2 of a sum of weights den * 2^m; a NaN is handed on as an infinite weight: the merge's maximum skips NaN.
__device__ __forceinline__ float log_weight(float m, float den) {
    return den == 0.f ? -INFINITY : (den <= FLT_MAX ? m + fast_log2(den) : INFINITY);
}

// Up to 28 chunks of a split pair are merged at once; more in groups of group_of(nch) and what is left, whose
// results, at most 16, are merged in turn.  (The whole call, at once / in groups: one sequence of 200k and
// one kv head, 444 chunks, 43.1 / 19.3 us; 32k and two heads 20.9 / 13.6; 32k and eight, 52 chunks, 20.2 / 19.2; 4k and
// eight, 32 chunks, 12.6 / 12.3; 3000 tokens, 24 chunks, 11.1 / 11.5.)
__device__ __forceinline__ int group_of(int nch) { return nch <= 28 ? nch : max(8, (nch + 15) / 16); }

// Partial results that are merged: number u lies in slot `head` (u = 0) or base + step * u.  The result goes to
// the outputs of hd's pair (to < 0) or to slot `to`.
struct Merge {
    int64_t head, base, to;
    int step, n;
};

// Merges this warp's share of each pass of kPassRows rows, kFlight chunks' loads in flight; called by the warp
// that finished the last of them.  (3 chunks of a short sequence, the whole call: 8.5 us with 4 in flight, 9.3
// with 16; 5 chunks 8.6 with 8, 9.1 with 16.)
template <bool BF16, int NT, int kFlight>
__device__ __forceinline__ void merge_share(const Params& p, const Header& hd, const Merge& mg, int warp, int lane) {
    using C = Cfg<NT>;
    for (int r0 = 0; r0 < p.rows; r0 += C::kPassRows) {
        const int share = min(C::kPassRows, p.rows - r0) * (kD / kWarps);
        for (int i = 4 * lane; i < share; i += 128) {
            const int e = r0 * kD + warp * share + i, r = e >> 7, d = e & (kD - 1);
            float m = -INFINITY, den = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
            for (int c0 = 0; c0 < mg.n; c0 += kFlight) {
                float lse[kFlight];
                float4 x[kFlight];
                float mx = m;
#pragma unroll
                for (int u = 0; u < kFlight; ++u) {
                    lse[u] = -INFINITY;
                    x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (c0 + u < mg.n) {
                        const int64_t slot = c0 + u == 0 ? mg.head : mg.base + mg.step * (c0 + u);
                        lse[u] = __ldcg(p.part_lse + (slot * kWarps + warp) * p.rows + r);
                        x[u] = __ldcg(reinterpret_cast<const float4*>(p.part_o + (slot * p.rows + r) * kD + d));
                    }
                }
#pragma unroll
                for (int u = 0; u < kFlight; ++u) mx = fmaxf(mx, lse[u]);
                if (mx == -INFINITY) continue;
                const float sc = fast_exp2(m - mx);
                den *= sc;
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[k] *= sc;
#pragma unroll
                for (int u = 0; u < kFlight; ++u) {
                    const float w = lse[u] == -INFINITY ? 0.f : fast_exp2(lse[u] - mx);
                    den += w;
                    acc[0] = fmaf(w, x[u].x, acc[0]);
                    acc[1] = fmaf(w, x[u].y, acc[1]);
                    acc[2] = fmaf(w, x[u].z, acc[2]);
                    acc[3] = fmaf(w, x[u].w, acc[3]);
                }
                m = mx;
            }
            const float inv = den == 0.f ? 0.f : __fdividef(1.f, den);
            if (mg.to < 0) {
                *reinterpret_cast<uint2*>(p.out + out_row(p, hd.b, hd.h, r) + d) =
                    make_uint2(pack2<BF16>(acc[0] * inv, acc[1] * inv), pack2<BF16>(acc[2] * inv, acc[3] * inv));
            } else {
                *reinterpret_cast<float4*>(p.part_o + (mg.to * p.rows + r) * kD + d) =
                    make_float4(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
                if (i == 0 || d == 0) p.part_lse[(mg.to * kWarps + warp) * p.rows + r] = log_weight(m, den);
            }
        }
    }
}

// What this warp of a CTA with an expired wait did not finish of the pairs that the CTA shares with others: NaN
// as its part (log_weight) and its header.  A call, and the plan made anew: inlined, or with the plan held over
// the loop, it takes registers from the loop (3 % of a decode call).
template <int NT>
__device__ __noinline__ void give_up(const Params& p, Smem<NT>& sm, int warp, int lane) {
    int length = 0, at = 0;
    for (int b = 0; b < p.batch; ++b) length += span_of(tiles_of(sm.lens[b])) * p.hkv;
    const int share = max(1, (length + int(gridDim.x) - 1) / int(gridDim.x));
    const int from = int(blockIdx.x) * share;
    for (int b = 0; b < p.batch && at < from + share; ++b) {
        const int nt = tiles_of(sm.lens[b]), span = span_of(nt);
        for (int h = 0; h < p.hkv && at < from + share; ++h, at += span) {
            if (nt == 0 || at + nt <= from) continue;
            const int first = at / share, nch = (at + nt - 1) / share - first + 1;
            const int side = int(blockIdx.x) == first ? 1 : 0;
            if (nch == 1 || sm.part[warp][side].nch != 0) continue;
            __syncwarp();
            if (lane < p.rows) p.part_lse[((2 * int64_t(blockIdx.x) + side) * kWarps + warp) * p.rows + lane] = INFINITY;
            if (lane == 0) sm.part[warp][side] = Header{b, h, first, nch};
            __syncwarp();
        }
    }
}

template <bool BF16, int NT>
__global__ void __launch_bounds__(kThreads, Cfg<NT>::kCtas) paged_attention_q4_kernel(const __grid_constant__ Params p) {
    using C = Cfg<NT>;
    extern __shared__ uint8_t smem_raw[];
    Smem<NT>& sm = *reinterpret_cast<Smem<NT>*>(smem_raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int cap = p.bt_width * p.block_size;  // tokens addressable through the block table

    if (tid == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&sm.full[s], 1);
            mbar_init(&sm.empty[s], kWarps);
        }
        mbar_init(&sm.cbar, kConsumers);
        sm.err = 0;
        fence_mbar_init();
    }

    // ---- plan: this CTA's run ------------------------------------------
    const int run = (p.batch + kConsumers - 1) / kConsumers;  // sequences per thread; off[] has every second
    int total;                                                // length of all pairs
    {
        int mine = 0, before = 0;
        if (warp < kWarps) {
            for (int b = tid * run; b < min((tid + 1) * run, p.batch); ++b) {
                const int ctx = min(max(p.context_lens[b], 0), cap);
                sm.lens[b] = ctx;
                mine += span_of(tiles_of(ctx));
            }
            before = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, before, o);
                if (lane >= o) before += y;
            }
            if (lane == 31) sm.red[warp] = before;
        }
        __syncthreads();
        total = 0;
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) before += sm.red[w];
            total += sm.red[w];
        }
        if (warp < kWarps && !(tid & 1)) sm.off[tid >> 1] = before - mine;
        total *= p.hkv;
        __syncthreads();
    }
    const int quota = max(1, (total + int(gridDim.x) - 1) / int(gridDim.x));
    const int begin = int(min(int64_t(blockIdx.x) * quota, int64_t(total))), end = min(begin + quota, total);

    if (warp == kWarps) {
        // ------------------------------------------------------------ producer
        if (begin >= end) return;
        // First pair of the run: its entry of off[] (the last that begins at or before it), then along the entry.
        static_assert(kConsumers / 2 == 64, "two entries per lane");
        const int entry = __popc(__ballot_sync(0xffffffffu, sm.off[lane] * p.hkv <= begin)) +
                          __popc(__ballot_sync(0xffffffffu, sm.off[32 + lane] * p.hkv <= begin)) - 1;
        if (lane == 0 && p.idle_producer != 1 && p.idle_producer != 2 + int(blockIdx.x)) {
            const uint64_t pol = l2_policy_evict_first();
            const uint32_t q_bytes = uint32_t(p.group) * kD * 2;  // one query token's rows of this kv head
            int b = 2 * entry * run, at = sm.off[entry] * p.hkv;  // `at`: where the current pair begins
            int ctx = sm.lens[b], nt = tiles_of(ctx);
            while (at + span_of(nt) * p.hkv <= begin) {
                at += span_of(nt) * p.hkv;
                ctx = sm.lens[++b];
                nt = tiles_of(ctx);
            }
            int h = (begin - at) / span_of(nt);
            at += h * span_of(nt);
            int t = begin - at;
            const int64_t head_bytes = int64_t(p.block_size) * kRecord, page_bytes = p.hkv * head_bytes;
            const int32_t* table = p.block_tables + b * p.bt_stride;
            int page = 0, off = 0;  // of tile t
            // The first tile of the next pair that has one, if it lies in this run.
            auto next_pair = [&] {
                t = page = off = 0;
                at += span_of(nt);
                if (at >= end) return;
                if (++h == p.hkv) {
                    h = 0;
                    do {
                        ctx = sm.lens[++b];
                        nt = tiles_of(ctx);
                    } while (nt == 0);
                    table = p.block_tables + b * p.bt_stride;
                }
            };
            if (t >= nt) {
                next_pair();
            } else if (t > 0) {
                page = t * kTile / p.block_size;
                off = t * kTile - page * p.block_size;
            }
            int blk = at + t < end ? table[page] : 0;  // loaded one tile ahead

            int stage = 0, qb = 0;
            uint32_t phase = 0;
            int fills = 0;
            bool ok = true;
            int first_flag = kFirst;
            while (at + t < end) {
                const int cur_b = b, cur_h = h, cur_at = at, cur_nt = nt;
                const int tile = t, tile_ctx = ctx, tile_off = off, tile_blk = blk;
                // Where the walk goes next.
                off += kTile;
                if (off == p.block_size) off = 0, ++page;
                const bool pair_end = ++t == nt;
                if (pair_end) next_pair();
                const bool more = at + t < end, last = pair_end || !more;
                if (more) blk = table[page];
                if (!mbar_wait(&sm.empty[stage], phase ^ 1, p.wait_ns)) {
                    ok = false;
                    break;
                }
                const bool in_cache = tile_blk >= 0 && tile_blk < p.num_blocks;
                mbar_expect_tx(&sm.full[stage],
                               (in_cache ? uint32_t(kStageBytes) : 0u) + (first_flag ? q_bytes * p.lq : 0u));
                if (in_cache) {
                    uint8_t* st = sm.stages[stage];
                    const int64_t o = tile_blk * page_bytes + cur_h * head_bytes + tile_off * kRecord;
                    bulk_load_hint(st, p.k + o, kKvBytes, &sm.full[stage], pol);
                    bulk_load_hint(st + kKvBytes, p.v + o, kKvBytes, &sm.full[stage], pol);
                }
                if (first_flag) {
                    const uint16_t* qsrc = p.q + int64_t(cur_b) * p.lq * p.q_stride + int64_t(cur_h) * p.group * kD;
                    for (int j = 0; j < p.lq; ++j)
                        bulk_load(sm.qbuf[qb] + j * q_bytes, qsrc + int64_t(j) * p.q_stride, q_bytes, &sm.full[stage]);
                }
                // What the warps need with the tile is written while it is on its way.
                *reinterpret_cast<int4*>(&sm.tile[stage]) = make_int4(
                    tile, first_flag | (last ? kLast : 0) | (in_cache ? 0 : kNoPage) | (qb ? kQBuf : 0), tile_ctx, 0);
                if (last) {
                    const int first = cur_at / quota;
                    *reinterpret_cast<int4*>(&sm.item[stage]) =
                        make_int4(cur_b, cur_h, first, (cur_at + cur_nt - 1) / quota - first + 1);
                }
                mbar_arrive(&sm.full[stage]);
                ++fills;
                if (++stage == kStages) { stage = 0; phase ^= 1; }
                first_flag = last ? kFirst : 0;
                if (last) qb ^= 1;
            }
            if (ok) {
                if (mbar_wait(&sm.empty[stage], phase ^ 1, p.wait_ns)) {
                    sm.tile[stage].tile = -1;  // sentinel: no more tiles
                    mbar_arrive(&sm.full[stage]);
                } else {
                    ok = false;
                }
            }
            if (!ok) {
                atomicOr(p.error, DEV_ERR_WAIT_EMPTY);
                // Error path: wait (bounded) for every copy still in flight before the CTA's
                // shared memory is released.
                for (int s = 0; s < kStages; ++s) {
                    if (fills <= s) break;
                    const int f = s + ((fills - 1 - s) / kStages) * kStages;
                    if (!mbar_wait(&sm.full[s], uint32_t((f / kStages) & 1), p.wait_ns)) atomicOr(p.error, DEV_ERR_WAIT_DRAIN);
                }
            }
        }
        __syncwarp();
        return;
    }

    // ---------------------------------------------------------------- consumers
    // Rows without a cached token (CUDA-graph padding) have no tiles and get a zero output.
    const int64_t row_vec = int64_t(p.lq) * p.hq * kD / 8;  // uint4 per batch row
    for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
        if (sm.lens[b] == 0) {
            uint4* o = reinterpret_cast<uint4*>(p.out) + b * row_vec;
            for (int64_t i = tid; i < row_vec; i += kConsumers) o[i] = make_uint4(0, 0, 0, 0);
        }
    }
    if (begin >= end) return;
    const int g = lane >> 2, c = lane & 3;
    const int tok_warp = warp * kWarpTokens;
    // Byte offsets in a sub-tile's records: the rows this lane hands to ldmatrix (token lane & 7, group
    // lane >> 3; the parameters of token `lane`, of both sub-tiles), and the parameters of token g.
    const uint32_t frag_off = uint32_t(lane & 7) * kRecord + (lane >> 3) * 16;
    const uint32_t par_off = uint32_t(g) * kRecord + q4::kParams;
    const uint32_t word_off = uint32_t(lane) * kRecord + q4::kParams;
    // Scores in units of 2^-24, which the minima start as the MMAs' result; fp16 sums of q do not go down to
    // that unit, and 16 rows would spill (131.5 us against 133.4 for the verify call): there they join last.
    constexpr bool kMinFirst = BF16 && NT == 1;
    constexpr uint32_t kLo = 0x000f000fu, kHi = 0x00f000f0u;
    if (lane < 2) sm.part[warp][lane].nch = 0;
    __syncwarp();
    int stage = 0;
    uint32_t phase = 0, cphase = 0;
    // Query rows 8 nt + 2 c + e: reference (log2), factor of the scores.  (What the loop can recompute is not held:
    // a limit per row and the reach that E allows cost 4 us of 271, and 2 of the verify call.)
    float r_ref[NT][2], f_row[NT][2];
    // B operands of row 8 nt + g: q (two steps of a group), sum(q) of group c in parts: (0, first), (0, second),
    // bf16 (0, first), (second, third).
    uint32_t qf[kGroups][NT][4], qs[NT][2];
    // O^T fragments (16 dims x 8 rows in units of 2^-24), and the product with the parameter words:
    // its row g is sum_t p * (half-word g), rows 8.. are sum_t p.
    float o[kGroups][2][NT][4], om[NT][4];
    float unit = 1.f;  // 2^-E of group g >> 1
    bool reading = false;            // the last combine's shared memory may still be read by other warps
    while (true) {
        // Exit decisions are warp-uniform (the lanes' waits can disagree at the limit).
        if (!__all_sync(0xffffffffu, mbar_wait(&sm.full[stage], phase, p.wait_ns))) {
            atomicOr(p.error, DEV_ERR_WAIT_FULL);
            *reinterpret_cast<volatile int32_t*>(&sm.err) = 1;
            break;
        }
        const int4 head = *reinterpret_cast<const int4*>(&sm.tile[stage]);
        const int tile = head.x, flags = head.y, ctx = head.z;
        // Votes tell the compiler that these branches are uniform.
        if (__any_sync(0xffffffffu, tile < 0)) break;
        if (__any_sync(0xffffffffu, flags & kFirst)) {
            // A sibling consumer warp that gave up will not reach the consumer barrier below.
            if (__any_sync(0xffffffffu, *reinterpret_cast<volatile int32_t*>(&sm.err) != 0)) break;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int row = 8 * nt + g;
                const uint8_t* qrow = sm.qbuf[flags & kQBuf ? 1 : 0] + row * kD * 2;
                float x[kGroups][8];
                float mx = 0.f;
#pragma unroll
                for (int j = 0; j < kGroups; ++j) {
                    uint4 w = make_uint4(0, 0, 0, 0);
                    if (row < p.rows) w = *reinterpret_cast<const uint4*>(qrow + (32 * j + 8 * c) * 2);
                    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        x[j][2 * i] = lo_f<BF16>(u[i]);
                        x[j][2 * i + 1] = hi_f<BF16>(u[i]);
                        mx = max3f(mx, fabsf(x[j][2 * i]), fabsf(x[j][2 * i + 1]));
                    }
                }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const int eq = mx > 0.f ? min(max((__float_as_int(mx) >> 23) - 127 - 3, -kExpMax), kExpMax) : 0;
                const float sc = exp2_int(-eq);
                float mine = 0.f;  // sum(q) of group c
#pragma unroll
                for (int j = 0; j < kGroups; ++j) {
                    float sum = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        x[j][i] *= sc;
                        sum += x[j][i];
                    }
                    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                    if (c == j) mine = sum;
                    qf[j][nt][0] = pack2<false>(x[j][0], x[j][1]);
                    qf[j][nt][1] = pack2<false>(x[j][2] * 0.0625f, x[j][3] * 0.0625f);
                    qf[j][nt][2] = pack2<false>(x[j][4], x[j][5]);
                    qf[j][nt][3] = pack2<false>(x[j][6] * 0.0625f, x[j][7] * 0.0625f);
                }
                const float sum_q = mine * (kMinFirst ? kCodeUnit : 1.f);
                if constexpr (BF16) {  // its 24 bits, eight at a time
                    const float first = __uint_as_float(__float_as_uint(sum_q) & 0xffff0000u), r = sum_q - first;
                    const float second = __uint_as_float(__float_as_uint(r) & 0xffff0000u);
                    qs[nt][0] = __float_as_uint(first);
                    qs[nt][1] = __byte_perm(__float_as_uint(second), __float_as_uint(r - second), 0x7632);
                } else {
                    split2(make_float2(0.f, sum_q), qs[nt][0], qs[nt][1]);
                }
                // Above zero even where that underflows (all scores are 0 then): a masked -inf stays one.
                const float fm = fmaxf(p.scale_log2 * exp2_int(eq) * (kMinFirst ? 1.f / kCodeUnit : 1.f), 1e-30f);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    f_row[nt][e] = __shfl_sync(0xffffffffu, fm, (2 * c + e) * 4);  // a lane of row rw
                    r_ref[nt][e] = kNone;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) om[nt][i] = 0.f;
#pragma unroll
                for (int j = 0; j < kGroups; ++j)
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[j][t][nt][e] = 0.f;
            }
            unit = exp2_int(kExpMax);
        }
        // Last token that row 8 nt + 2 c + e sees.  Padding rows see the whole context: only rows that exist mask.
        auto lim = [&](int nt, int e) {
            const int rw = 8 * nt + 2 * c + e;
            return rw < p.rows ? ctx - p.lq + ((rw * p.group_inv) >> 16) : ctx - 1;
        };
        bool wrote = false;
        {
            // Records past the context may hold anything (a NaN scale times a probability of 0 is
            // NaN), a page outside the cache was not loaded: both read as zeros.
            const int left = ctx - (tile * kTile + tok_warp);
            const int first = (flags & kNoPage) ? 0 : left;
            if (__any_sync(0xffffffffu, left > 0 && first < kWarpTokens)) {
                for (int i = lane; i < (kWarpTokens - first) * (kRecord / 16); i += 32) {
                    uint8_t* at = sm.stages[stage] + (tok_warp + first) * kRecord + i * 16;
                    *reinterpret_cast<uint4*>(at) = make_uint4(0, 0, 0, 0);
                    *reinterpret_cast<uint4*>(at + kKvBytes) = make_uint4(0, 0, 0, 0);
                }
                wrote = true;
                __syncwarp();
            }
        }
#pragma unroll 1
        for (int sub = 0; sub < kWarpTokens; sub += 32) {
            const int tok_base = tile * kTile + tok_warp + sub;
            if (__any_sync(0xffffffffu, tok_base >= ctx)) break;
            // Two copies of the step, so that the common one is straight code: EDGE is a step that reaches past
            // some row's last visible token.
            auto step = [&](auto edge) {
            constexpr bool EDGE = decltype(edge)::value;
            uint8_t* kb = sm.stages[stage] + (tok_warp + sub) * kRecord;
            uint8_t* vb = kb + kKvBytes;
            // ---- scores x (times f_row: log2): codes and minima of S^T = K Q^T ----
            float x[2][NT][4];  // sub-tile of 16: token g (+ 8 for e >= 2), rows 8 nt + 2 c, 2 c + 1
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint8_t* ks = kb + u * 16 * kRecord;
                uint32_t kw[2][kGroups];  // word c of token g (g + 8)
                ldsm_x4(kw[0][0], kw[0][1], kw[0][2], kw[0][3], smem_u32(ks) + frag_off);
                ldsm_x4(kw[1][0], kw[1][1], kw[1][2], kw[1][3], smem_u32(ks) + frag_off + 8 * kRecord);
                const uint4 pa4 = *reinterpret_cast<const uint4*>(ks + par_off);
                const uint4 pb4 = *reinterpret_cast<const uint4*>(ks + par_off + 8 * kRecord);
                const uint32_t pa[4] = {pa4.x, pa4.y, pa4.z, pa4.w}, pb[4] = {pb4.x, pb4.y, pb4.z, pb4.w};
                uint32_t a[4];  // word c of the parameters of tokens g, g + 8; again, or (bf16) their minima twice
                auto load_words = [&] {
                    ldsm_x2(a[0], a[1], smem_u32(ks) + word_off);
                    a[2] = BF16 ? __byte_perm(a[0], 0, 0x3232) : a[0];
                    a[3] = BF16 ? __byte_perm(a[1], 0, 0x3232) : a[1];
                };
                if constexpr (kMinFirst) {
                    load_words();
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma_zero<BF16>(x[u][nt], a, qs[nt][0], qs[nt][1]);
                }
#pragma unroll
                for (int j = 0; j < kGroups; ++j) {
                    const uint32_t wa = kw[0][j], wb = kw[1][j], wa8 = wa >> 8, wb8 = wb >> 8;
                    const uint32_t a0[4] = {wa & kLo, wb & kLo, wa & kHi, wb & kHi};
                    const uint32_t a1[4] = {wa8 & kLo, wb8 & kLo, wa8 & kHi, wb8 & kHi};
                    const float sa = lo_f<BF16>(pa[j]), sb = lo_f<BF16>(pb[j]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float acc[4];
                        mma_zero<false>(acc, a0, qf[j][nt][0], qf[j][nt][1]);
                        mma<false>(acc, a1, qf[j][nt][2], qf[j][nt][3]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float sc = e < 2 ? sa : sb;
                            x[u][nt][e] = !kMinFirst && j == 0 ? sc * acc[e] : fmaf(sc, acc[e], x[u][nt][e]);
                        }
                    }
                }
                if constexpr (!kMinFirst) {
                    load_words();
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float xm[4];
                        mma_zero<BF16>(xm, a, qs[nt][0], qs[nt][1]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[u][nt][e] = fmaf(x[u][nt][e], 1.f / kCodeUnit, xm[e]);
                    }
                }
            }
            // ---- masks; references ----
            if constexpr (EDGE) {
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (tok_base + 16 * u + g + (e >> 1) * 8 > lim(nt, e & 1)) x[u][nt][e] = -INFINITY;
            }
            float y_max = -INFINITY;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    y_max = fmaxf(y_max, fmaf(max3f(fmaxf(x[0][nt][e], x[0][nt][2 + e]), x[1][nt][e], x[1][nt][2 + e]),
                                              f_row[nt][e], -r_ref[nt][e]));
            // Half-word g of the value parameters of tokens 8 i + 2 c, 2 c + 1.
            uint32_t w[4];
            ldsm_x4_t(w[0], w[1], w[2], w[3], smem_u32(vb) + word_off);
            const uint32_t wt = max_abs<BF16>(max_abs<BF16>(w[0], w[1]), max_abs<BF16>(w[2], w[3]));
            // max(16 s, |m|) of group g >> 1, of those (NaNs apart).
            float top = fmaxf(fabsf(lo_f<BF16>(wt)), fabsf(hi_f<BF16>(wt))) * (lane & 4 ? 1.f : 16.f);
            if (__any_sync(0xffffffffu, y_max > kLazyMax || top * unit > kReach)) {
                // Rare: raise the groups' E to the value parameters of this tile, the rows' maxima to its scores.
#pragma unroll
                for (int sh = 1; sh <= 4; sh <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, sh));
                float drop = 1.f;  // 2^-(rise of E)
                if (top * unit > kReach) {
                    const int old = 127 - (__float_as_int(unit) >> 23);  // E
                    const int en = min(max((__float_as_int(top) >> 23) - 127 - kUnitBits, old), kExpMax);
                    drop = exp2_int(old - en);
                    unit = exp2_int(-en);
                }
                float alpha[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float tm = max3f(fmaxf(x[0][nt][e], x[0][nt][2 + e]), x[1][nt][e], x[1][nt][2 + e]);
#pragma unroll
                        for (int sh = 4; sh <= 16; sh <<= 1) tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, sh));
                        tm *= f_row[nt][e];
                        const float ro = r_ref[nt][e], rn = fmaxf(ro, tm == -INFINITY ? kNone : tm - kTop);
                        alpha[nt][e] = ro == kNone ? 0.f : fast_exp2(ro - rn);
                        r_ref[nt][e] = rn;
                    }
                // An item's first step has nothing to scale: skipped for up to 16 rows (verify 129.9 -> 127.5 us).  For up
                // to 8 the branch costs registers that spill (decode of 512 sequences 267.1 us without, 271.5 with).
                if (NT == 1 || !__any_sync(0xffffffffu, flags & kFirst)) {
                    float drops[kGroups];
#pragma unroll
                    for (int j = 0; j < kGroups; ++j) drops[j] = __shfl_sync(0xffffffffu, drop, 8 * j);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            om[nt][e] *= alpha[nt][e] * drop;
                            om[nt][2 + e] *= alpha[nt][e];
#pragma unroll
                            for (int j = 0; j < kGroups; ++j)
#pragma unroll
                                for (int t = 0; t < 2; ++t) {
                                    o[j][t][nt][e] *= alpha[nt][e] * drops[j];
                                    o[j][t][nt][2 + e] *= alpha[nt][e] * drops[j];
                                }
                        }
                }
            }
            if constexpr (EDGE) {
                // A stored non-finite value (s = m = NaN) counts for the rows that see its token only: it
                // becomes a NaN of their sums here, and a zero as an operand below.
                const uint4 look = *reinterpret_cast<const uint4*>(vb + word_off);  // of token `lane`
                const uint32_t lw[4] = {look.x, look.y, look.z, look.w};
#pragma unroll
                for (int j = 0; j < kGroups; ++j) {
                    const bool mine = !(fabsf(lo_f<BF16>(lw[j])) <= FLT_MAX && fabsf(hi_f<BF16>(lw[j])) <= FLT_MAX);
                    uint32_t bad = __ballot_sync(0xffffffffu, mine);
                    for (; bad; bad &= bad - 1) {
                        const int t = tok_base + __ffs(bad) - 1;
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 2; ++e)
                                if (g == 2 * j + 1 && t <= lim(nt, e)) om[nt][e] = __int_as_float(0x7fffffff);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint8_t* vs = vb + u * 16 * kRecord;
                // P in fp16, as B operands: lane (g, c) holds row g of tokens 2 c, 2 c + 1 (+ 8); for fp16
                // models also what the rounding left.
                uint32_t pb[NT][2], pl[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float2 y = make_float2(fast_exp2(fmaf(x[u][nt][2 * i], f_row[nt][0], -r_ref[nt][0])),
                                                     fast_exp2(fmaf(x[u][nt][2 * i + 1], f_row[nt][1], -r_ref[nt][1])));
                        if constexpr (BF16) {
                            pb[nt][i] = transpose8(pack2<false>(y.x, y.y));
                        } else {
                            uint32_t hi, lo;
                            split2(y, hi, lo);
                            pb[nt][i] = transpose8(hi);
                            pl[nt][i] = transpose8(lo);
                        }
                    }
                // Half-word g of their parameters, times 2^-E in fp16; ones.
                uint32_t pt[4];
                ldsm_x2_t(pt[0], pt[2], smem_u32(vs) + word_off);
                pt[1] = pt[3] = 0x3c003c00u;
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    if constexpr (EDGE) pt[i] = finite2<BF16>(pt[i]);
                    pt[i] = pack2<false>(lo_f<BF16>(pt[i]) * unit, hi_f<BF16>(pt[i]) * unit);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    mma<false>(om[nt], pt, pb[nt][0], pb[nt][1]);
                    if constexpr (!BF16) mma<false>(om[nt], pt, pl[nt][0], pl[nt][1]);
                }
                // ---- O^T += V^T (P s)^T ----
                uint32_t vw[2][kGroups];  // half-word g of tokens 2 c, 2 c + 1 (+ 8)
                ldsm_x4_t(vw[0][0], vw[0][1], vw[0][2], vw[0][3], smem_u32(vs) + frag_off);
                ldsm_x4_t(vw[1][0], vw[1][1], vw[1][2], vw[1][3], smem_u32(vs) + frag_off + 8 * kRecord);
#pragma unroll
                for (int j = 0; j < kGroups; ++j) {
                    // The scales of group j: half-word 2 j, from the lanes of row 2 j.
                    uint32_t b[NT][2], bl[NT][2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t sc = __shfl_sync(0xffffffffu, pt[2 * i], 8 * j + c);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            b[nt][i] = mul_f16x2(pb[nt][i], sc);
                            // What rounding p s to fp16 left (the fused residual is exact).
                            if constexpr (!BF16)
                                bl[nt][i] = fma_f16x2(pl[nt][i], sc, fma_f16x2(pb[nt][i], sc, b[nt][i] ^ 0x80008000u));
                        }
                    }
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        // Bytes n + 16 n' (n' the next nibble) and their low nibbles n: one operation each.
                        const uint32_t w0 = t ? __byte_perm(vw[0][j], 0, 0x4341) : vw[0][j] & 0x00ff00ffu;
                        const uint32_t w1 = t ? __byte_perm(vw[1][j], 0, 0x4341) : vw[1][j] & 0x00ff00ffu;
                        const uint32_t a[4] = {w0 & kLo, w0, w1 & kLo, w1};
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma<false>(o[j][t][nt], a, b[nt][0], b[nt][1]);
                            if constexpr (!BF16) mma<false>(o[j][t][nt], a, bl[nt][0], bl[nt][1]);
                        }
                    }
                }
            }
            };
            if (__any_sync(0xffffffffu, tok_base + 31 > ctx - p.lq)) step(std::true_type{});
            else step(std::false_type{});
        }
        if (wrote) fence_proxy_async_smem();
        const bool item_end = __any_sync(0xffffffffu, flags & kLast);
        Header hd{0, 0, 0, 0};
        if (item_end) hd = sm.item[stage];
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.empty[stage]);
        if (++stage == kStages) { stage = 0; phase ^= 1; }
        if (!item_end) continue;

        // ---- combine the warps' states of this item ----
        // O = 2^E (2^24 o + sum p m); n' is a sixteenth of the byte's sum less the low nibble's.
        float back[kGroups];  // 2^E
#pragma unroll
        for (int j = 0; j < kGroups; ++j)
            back[j] = __shfl_sync(0xffffffffu, __int_as_float(0x7f000000 - __float_as_int(unit)), 8 * j);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int j = 0; j < kGroups; ++j) {
                    const float mj = __shfl_sync(0xffffffffu, om[nt][e], (2 * j + 1) * 4 + c);
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        o[j][t][nt][2 + e] = fmaf(o[j][t][nt][2 + e] - o[j][t][nt][e], 1048576.f, mj) * back[j];
                        o[j][t][nt][e] = fmaf(o[j][t][nt][e], 16777216.f, mj) * back[j];
                    }
                }
        // Dimension of o[j][t][.][e] for e < 2; e >= 2 is the next nibble, two dimensions on.
        const int d0 = 8 * (g >> 1) + (g & 1);
        const bool single = hd.nch == 1;
        const int64_t slot = 2 * int64_t(blockIdx.x) + (int(blockIdx.x) == hd.first ? 1 : 0);
        bool ok = true;
#pragma unroll
        for (int r0 = 0; r0 < 8 * NT; r0 += C::kPassRows) {
            if (r0 >= p.rows || !ok) break;
            const int nr = min(C::kPassRows, p.rows - r0);
            if (reading) ok = consumer_wait(&sm.cbar, cphase, p.wait_ns);
            if (!ok) break;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int r = 8 * nt + 2 * c + e - r0;
                    if (r >= 0 && r < nr) {
                        if (g == 0) {
                            sm.cm[warp][r] = r_ref[nt][e];
                            sm.cl[warp][r] = om[nt][2 + e];
                        }
#pragma unroll
                        for (int j = 0; j < kGroups; ++j)
#pragma unroll
                            for (int t = 0; t < 2; ++t) {
                                float* cp = &sm.co[warp][r][32 * j + 4 * t + d0];
                                cp[0] = o[j][t][nt][e];
                                cp[2] = o[j][t][nt][2 + e];
                            }
                    }
                }
            mbar_arrive(&sm.cbar);
            ok = consumer_wait(&sm.cbar, cphase, p.wait_ns);
            if (!ok) break;
            // A quarter of the pass's elements each, two neighbours per lane and round.
            const int n = nr * (kD / kWarps);
            for (int i = 2 * lane; i < n; i += 64) {
                const int el = warp * n + i, r = el >> 7, d = el & (kD - 1);
                float M = sm.cm[0][r];
#pragma unroll
                for (int w = 1; w < kWarps; ++w) M = fmaxf(M, sm.cm[w][r]);
                float den = 0.f, a0 = 0.f, a1 = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float sc = fast_exp2(sm.cm[w][r] - M);
                    den = fmaf(sm.cl[w][r], sc, den);
                    a0 = fmaf(sm.co[w][r][d], sc, a0);
                    a1 = fmaf(sm.co[w][r][d + 1], sc, a1);
                }
                const float inv = den == 0.f ? 0.f : __fdividef(1.f, den);  // 0: the row sees no token of this item
                const int row = r0 + r;
                if (single)
                    *reinterpret_cast<uint32_t*>(p.out + out_row(p, hd.b, hd.h, row) + d) = pack2<BF16>(a0 * inv, a1 * inv);
                else
                    *reinterpret_cast<float2*>(p.part_o + (slot * p.rows + row) * kD + d) = make_float2(a0 * inv, a1 * inv);
            }
            if (!single && lane < nr) {
                float M = sm.cm[0][lane];
#pragma unroll
                for (int w = 1; w < kWarps; ++w) M = fmaxf(M, sm.cm[w][lane]);
                float den = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) den = fmaf(sm.cl[w][lane], fast_exp2(sm.cm[w][lane] - M), den);
                p.part_lse[(slot * kWarps + warp) * p.rows + r0 + lane] = log_weight(M, den);
            }
            mbar_arrive(&sm.cbar);
            reading = true;
        }
        if (!ok) {
            atomicOr(p.error, DEV_ERR_WAIT_PEER);
            *reinterpret_cast<volatile int32_t*>(&sm.err) = 1;
            break;
        }
        if (!single && lane == 0) sm.part[warp][slot & 1] = hd;
    }

    // A CTA with an expired wait counts all the same for the split pairs it shares, so that the counters are
    // zero again for the next call.
    __syncwarp();
    if (__any_sync(0xffffffffu, *reinterpret_cast<volatile int32_t*>(&sm.err) != 0)) give_up<NT>(p, sm, warp, lane);

    // The run's partial items (its first and its last), after the loop so that the merge's registers are
    // not held beside it: publish this warp's share of each (one releasing count per warp, cumulative over the
    // warp barrier), then count it; the last chunk's warp of this number merges the share.  Groups are
    // counted and merged in what belongs to their second chunk's CTA, which has no other item.
    auto arrive_last = [&](int cta, int n) {
        __syncwarp();
        int last = 0;
        if (lane == 0) {
            int32_t* counter = &p.counters[cta * kWarps + warp];
            last = atomic_inc_acq_rel(counter) == n - 1;
            if (last) *counter = 0;
        }
        last = __shfl_sync(0xffffffffu, last, 0);
        __syncwarp();
        return last;
    };
    auto merge = [&](const Header& hd, const Merge& mg) {
        if (mg.n <= 4) merge_share<BF16, NT, 4>(p, hd, mg, warp, lane);
        else if (mg.n <= 8) merge_share<BF16, NT, 8>(p, hd, mg, warp, lane);
        else merge_share<BF16, NT, 16>(p, hd, mg, warp, lane);
    };
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
        const Header hd = sm.part[warp][i];
        if (hd.nch == 0) continue;
        Merge mg{2 * int64_t(hd.first) + 1, 2 * int64_t(hd.first), -1, 2, hd.nch};
        const int size = group_of(hd.nch), groups = hd.nch / size;
        if (groups > 1) {
            const int grp = min((int(blockIdx.x) - hd.first) / size, groups - 1), c0 = grp * size, cta = hd.first + c0 + 1;
            const int n = grp == groups - 1 ? hd.nch - c0 : size;
            if (!arrive_last(cta, n)) continue;
            const int64_t at = 2 * int64_t(hd.first + c0);
            merge(hd, Merge{at + (grp == 0), at, 2 * int64_t(cta) + 1, 2, n});
            const int64_t to = 2 * int64_t(hd.first + 1) + 1;
            mg = Merge{to, to, -1, 2 * size, groups};
        }
        if (!arrive_last(hd.first, mg.n)) continue;
        merge(hd, mg);
    }
}

template <bool BF16, int NT>
void launch(const Params& prm, int ctas, cudaStream_t s) {
    // The shared-memory limit is set once per device (a call of its own costs the host as much as the
    // argument checks); setting it twice does no harm.
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64 || !(done.load(std::memory_order_relaxed) >> dev & 1)) {
        ensure_smem_attr((const void*)paged_attention_q4_kernel<BF16, NT>, int(sizeof(Smem<NT>)));
        if (dev < 64) done.fetch_or(uint64_t(1) << dev, std::memory_order_relaxed);
    }
    paged_attention_q4_kernel<BF16, NT><<<ctas, kThreads, sizeof(Smem<NT>), s>>>(prm);
}

}  // namespace
}  // namespace pq4
}  // namespace b200

extern "C" size_t b200_paged_attention_q4_workspace_size(int32_t query_len, int32_t group_size) {
    using namespace b200::pq4;
    if (query_len < 1 || group_size < 1) return 0;
    const int64_t rows = int64_t(query_len) * group_size;
    return rows > 16 ? 0 : workspace_bytes(int(rows));
}

extern "C" int32_t b200_stream_capture_id(void* stream, uint64_t* id) {
    using namespace b200;
    clear_error();
    B200_REQUIRE(id, "stream_capture_id: null pointer");
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    unsigned long long capture = 0;
    B200_CUDA_TRY(cudaStreamGetCaptureInfo(static_cast<cudaStream_t>(stream), &status, &capture));
    *id = status == cudaStreamCaptureStatusActive ? capture : 0;
    return B200_OK;
}

extern "C" int32_t b200_paged_attention_q4(void* out, const void* q, int64_t q_stride_token, const void* k_cache,
                                           const void* v_cache, int32_t num_blocks, int32_t block_size,
                                           const int32_t* block_tables, int64_t block_table_stride,
                                           int32_t block_table_width, const int32_t* context_lens, int32_t batch,
                                           int32_t query_len, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                           float softmax_scale, int32_t dtype, void* workspace, size_t workspace_size,
                                           void* stream) {
    using namespace b200;
    using namespace b200::pq4;
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
                     block_table_stride >= 0,
                 "paged_attention_q4: block table of %d entries, stride %lld out of range", block_table_width,
                 (long long)block_table_stride);
    if ((int64_t(block_table_width) * (block_size / kTile) + kPairCost) * batch > INT32_MAX / 2 / num_kv_heads)
        return fail(B200_ERR_UNSUPPORTED, "paged_attention_q4: %d tables of %d blocks of %d tokens", batch,
                    block_table_width, block_size);
    auto al16 = [](const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15) == 0; };
    B200_REQUIRE(q_stride_token >= int64_t(num_heads) * head_dim && q_stride_token % 8 == 0 && al16(q) && al16(out) &&
                     al16(k_cache) && al16(v_cache),
                 "paged_attention_q4: q, out and the caches must be 16-byte aligned, q token stride (%lld) a multiple of 8 "
                 "and at least Hq*D",
                 (long long)q_stride_token);
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) ||
        workspace_size < workspace_bytes(int(rows)))
        return fail(B200_ERR_WORKSPACE, "paged_attention_q4: workspace missing, unaligned or smaller than %zu bytes",
                    workspace_bytes(int(rows)));

    const int ctas = grid_ctas(int(rows));
    Params prm;
    prm.q = static_cast<const uint16_t*>(q);
    prm.q_stride = q_stride_token;
    prm.out = static_cast<uint16_t*>(out);
    prm.k = static_cast<const uint8_t*>(k_cache);
    prm.v = static_cast<const uint8_t*>(v_cache);
    prm.block_tables = block_tables;
    prm.bt_stride = block_table_stride;
    prm.bt_width = block_table_width;
    prm.context_lens = context_lens;
    prm.batch = batch;
    prm.lq = query_len;
    prm.hq = num_heads;
    prm.hkv = num_kv_heads;
    prm.group = group;
    prm.rows = int32_t(rows);
    prm.block_size = block_size;
    prm.num_blocks = num_blocks;
    prm.group_inv = (65536 + group - 1) / group;
    prm.scale_log2 = softmax_scale * 1.4426950408889634f;
    char* ws = static_cast<char*>(workspace);
    prm.error = reinterpret_cast<int32_t*>(ws) + 2;
    prm.counters = reinterpret_cast<int32_t*>(ws + kCtrlBytes);
    prm.part_o = reinterpret_cast<float*>(ws + fixed_bytes());
    prm.part_lse = prm.part_o + size_t(2) * ctas * rows * kD;
    take_test_hook(&prm.wait_ns, &prm.idle_producer);

    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == B200_BF16) {
        if (rows > 8) launch<true, 2>(prm, ctas, s);
        else launch<true, 1>(prm, ctas, s);
    } else {
        if (rows > 8) launch<false, 2>(prm, ctas, s);
        else launch<false, 1>(prm, ctas, s);
    }
    B200_CUDA_TRY(cudaGetLastError());
    return B200_OK;
}
