// Work decomposition of the paged attention kernels (one plan for the 16-bit and the 4-bit cache).
//
// A work item is (sequence b, kv head h, chunk c): up to `chunk` tiles of 128 cached tokens of
// one kv head.  Every CTA plans the chunks from context_lens on the device, items are claimed
// dynamically, and the chunks of a split sequence are merged by the CTA that finishes the last one.
#pragma once

#include "common.cuh"

namespace b200 {
namespace pa {

constexpr int kTile = 128;                   // tokens per stage
constexpr int kD = 128;
constexpr int kConsumerWarps = 8;
constexpr int kConsumers = kConsumerWarps * 32;
constexpr int kThreads = kConsumers + 32;
constexpr int kMaxBatch = 2048;
constexpr int kCounterSlots = 65536;
constexpr int kCtrlWords = 64;               // [0] next item, [1] finished CTAs, [2] error word
constexpr size_t kFixedBytes = kCtrlWords * 4 + size_t(kCounterSlots) * 4;
constexpr int kWaves = 3;
constexpr int kChunkMaxTiles = 32;           // at most 4096 tokens per item
constexpr int kRemBits = 12;                 // packed offsets: full-chunk offset << 12 | remainder offset
constexpr int kClaimAhead = 1;               // tiles before an item's end at which the next one is claimed
constexpr float kLazyMax = 8.f;              // log2 headroom before a row's running maximum is raised

struct Header {
    int32_t item, b, h, tile, flags, ctx, nchunks, slot0;
};
enum : int32_t { kFirst = 1, kLast = 2 };

struct Params {
    const uint16_t* q;
    int64_t q_stride;
    uint16_t* out;
    const int32_t* block_tables;
    int32_t bt_stride;
    int32_t bt_width;  // entries of a row (the 16-bit kernel takes rows as wide as their stride)
    const int32_t* context_lens;
    int32_t batch, lq, hq, hkv, group, rows, block_size, num_blocks;
    float scale_log2;
    uint64_t wait_ns;  // limit of every wait (kWaitLimitNs; shorter under the idle-producer test)
    int32_t idle_producer;  // test hook: the producer issues nothing, so the consumers' first wait runs out
    int32_t* ctrl;
    int32_t* counters;
    float* part_o;    // [max_items][rows][kD]
    float* part_lse;  // [max_items][rows]
    int32_t max_items;
};

// Wait limit and idle-producer flag of the next launch on this host thread (b200_testing_idle_producer).
void apply_test_hook(Params& prm);

// Block-wide exclusive scan of one int per thread; returns the exclusive
// prefix and writes the total to *total.  Uses red[] (one slot per warp).
__device__ __forceinline__ int block_exclusive_scan(int v, int* red, int* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) red[warp] = x;
    __syncthreads();
    int base = 0, tot = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
        if (w < warp) base += red[w];
        tot += red[w];
    }
    __syncthreads();
    *total = tot;
    return base + x - v;
}

// Barrier of the consumer threads, bounded: each arrives (release) and polls
// the phase (acquire) for at most limit_ns.  Returns false, for the whole
// warp alike, when the wait of any of its lanes ran out.
__device__ __forceinline__ bool consumer_sync(uint64_t* bar, uint32_t& phase, uint64_t limit_ns) {
    mbar_arrive(bar);
    const bool ok = mbar_wait_spin(bar, phase, limit_ns);
    phase ^= 1;
    return __all_sync(0xffffffffu, ok);
}

// Chunk layout of one sequence: `full` items in the first region (chunks of
// `chunk` tiles, the last of them possibly a remainder of at least half a
// chunk) and `rem` (0 or 1) short remainder in the second.
struct SeqChunks {
    int nt, full, rem;
};

// A sequence of nt tiles is cut into chunks of `chunk` tiles and a shorter remainder.  Items
// are numbered in two regions: first every sequence's full chunks together with its remainder
// when that is at least half a chunk ("full" count), then the short remainders ("rem"), so that
// the smallest items come last and the end of a launch is made of them.
__device__ __forceinline__ SeqChunks tile_chunks(int nt, int64_t chunk) {
    SeqChunks s;
    s.nt = nt;
    s.full = int(nt / chunk);
    const int64_t rt = nt - int64_t(s.full) * chunk;
    const bool big = rt > 0 && 2 * rt >= chunk;
    s.full += big ? 1 : 0;
    s.rem = (rt > 0 && !big) ? 1 : 0;
    return s;
}

__device__ __forceinline__ SeqChunks seq_chunks(int ctx, int cap, int64_t chunk) {
    ctx = min(ctx, cap);
    return tile_chunks(ctx > 0 ? (ctx + kTile - 1) / kTile : 0, chunk);
}

// Metadata of one claimed work item.  The producer fetches it one item
// ahead, so that its dependent global loads (context length, block ids)
// overlap the TMA traffic of the current item.
constexpr int kPrefetchPages = 4;
struct ItemMeta {
    int item, b, h, c, nchunks, ctx, t0, slot0, page0;
    int blk[kPrefetchPages];
};

// Partial-output slot (chunk index, before the x Hkv + h) of chunk c of
// sequence b: first-region chunks are numbered first, short remainders after them.
__device__ __forceinline__ int chunk_slot(int packed_off, int c, int full, int total_full) {
    return c < full ? (packed_off >> kRemBits) + c : total_full + (packed_off & ((1 << kRemBits) - 1));
}

__device__ __forceinline__ void fetch_meta(ItemMeta& m, int item, const Params& p, const int32_t* off,
                                           int total_full, int64_t chunk, int cap) {
    m.item = item;
    const int cg = item / p.hkv;
    m.h = item - cg * p.hkv;
    int blo = 0, bhi = p.batch;  // largest b whose offset (in the chunk's group) is <= cg
    if (cg < total_full) {
        while (bhi - blo > 1) {
            const int mid = (blo + bhi) >> 1;
            if ((off[mid] >> kRemBits) <= cg) blo = mid; else bhi = mid;
        }
    } else {
        const int r = cg - total_full;
        while (bhi - blo > 1) {
            const int mid = (blo + bhi) >> 1;
            if ((off[mid] & ((1 << kRemBits) - 1)) <= r) blo = mid; else bhi = mid;
        }
    }
    m.b = blo;
    m.ctx = p.context_lens[blo];
    const SeqChunks sc = seq_chunks(m.ctx, cap, chunk);
    m.c = cg < total_full ? cg - (off[blo] >> kRemBits) : sc.full;
    m.nchunks = sc.full + sc.rem;
    m.slot0 = off[blo];
    m.t0 = int(m.c * chunk);
    m.page0 = (m.t0 * kTile) / p.block_size;
    const int32_t* bt = p.block_tables + int64_t(blo) * p.bt_stride;
#pragma unroll
    for (int j = 0; j < kPrefetchPages; ++j) m.blk[j] = bt[min(m.page0 + j, p.bt_width - 1)];
}

// What a CTA needs to know of the plan; the chunk offsets themselves are in its shared memory.
struct Plan {
    int cap;            // tokens addressable through the block table
    int64_t chunk;      // tiles per chunk
    int total_full;     // chunks of the first region
    int total_items;
};

// Plans the call: tiles per sequence, chunk length, chunk offsets (off[batch + 1], red one slot
// per warp, both in shared memory).  Ends with a block barrier.
__device__ __forceinline__ Plan plan_items(const Params& p, int32_t* off, int32_t* red) {
    const int tid = threadIdx.x;
    Plan pl;
    pl.cap = p.bt_width * p.block_size;  // tokens addressable through the block table
    const int seg = (p.batch + kThreads - 1) / kThreads;
    const int lo = min(tid * seg, p.batch), hi = min(lo + seg, p.batch);
    int my_tiles = 0;
    for (int b = lo; b < hi; ++b) {
        const int nt = seq_chunks(p.context_lens[b], pl.cap, 1).nt;
        off[b] = nt;  // this thread's sequences only; replaced by their offsets below
        my_tiles += nt;
    }
    int total_tiles = 0;
    block_exclusive_scan(my_tiles, red, &total_tiles);
    int64_t& chunk = pl.chunk;
    {
        const int64_t want = int64_t(gridDim.x) * kWaves;
        chunk = (int64_t(total_tiles) * p.hkv + want - 1) / want;
        chunk = chunk < 1 ? 1 : (chunk > kChunkMaxTiles ? kChunkMaxTiles : chunk);
        const int64_t budget = p.max_items / p.hkv;
        if (budget > p.batch) {
            const int64_t need = (int64_t(total_tiles) + (budget - p.batch) - 1) / (budget - p.batch);
            if (need > chunk) chunk = need;
        } else {
            chunk = int64_t(1) << 30;
        }
        // First-region offsets are packed into 31 - kRemBits bits (full chunks, plus at most one
        // remainder per sequence).
        const int64_t max_full = (int64_t(1) << (31 - kRemBits)) - 1 - kMaxBatch;
        if (int64_t(total_tiles) / chunk > max_full) chunk = (int64_t(total_tiles) + max_full - 1) / max_full;
    }
    // Both offsets in one scan of the packed count full << kRemBits | rem: the remainder
    // counts sum to at most the batch (< 2^kRemBits), so no carry reaches the full part.
    int my_packed = 0;
    for (int b = lo; b < hi; ++b) {
        const SeqChunks sc = tile_chunks(off[b], chunk);
        my_packed += (sc.full << kRemBits) + sc.rem;
    }
    int total_packed = 0;
    int opacked = block_exclusive_scan(my_packed, red, &total_packed);
    for (int b = lo; b < hi; ++b) {
        const SeqChunks sc = tile_chunks(off[b], chunk);
        off[b] = opacked;
        opacked += (sc.full << kRemBits) + sc.rem;
    }
    pl.total_full = total_packed >> kRemBits;
    const int total_rem = total_packed & ((1 << kRemBits) - 1);
    if (tid == 0) off[p.batch] = total_packed;
    __syncthreads();
    pl.total_items = (pl.total_full + total_rem) * p.hkv;
    return pl;
}

// Merges the chunks of a split (sequence, kv head) and writes its output rows; called by all
// consumer threads of the CTA that finished the last chunk.
template <bool BF16>
__device__ __forceinline__ void merge_chunks(const Params& p, const Header& hd, const Plan& pl, int tid) {
    const int nch = hd.nchunks;
    const int nel = p.rows * kD;
    const int full = nch - (seq_chunks(hd.ctx, pl.cap, pl.chunk).rem);
    // One pass over the chunks, four at a time: every thread merges the
    // partials of two output elements at once with a running maximum of the
    // chunks' log-sum-exps (base 2), the sixteen loads of a group in flight.
    for (int e0 = 2 * tid; e0 < nel; e0 += 2 * kConsumers) {
        const int r = e0 >> 7, d = e0 & (kD - 1);  // d even: (d, d + 1) in one row
        float mrun = -INFINITY, den = 0.f, acc0 = 0.f, acc1 = 0.f;
        for (int c0 = 0; c0 < nch; c0 += 4) {
            float lse[4];
            float2 x[4];
#pragma unroll
            for (int cc = 0; cc < 4; ++cc) {
                if (c0 + cc < nch) {
                    const int64_t it =
                        int64_t(chunk_slot(hd.slot0, c0 + cc, full, pl.total_full)) * p.hkv + hd.h;
                    lse[cc] = __ldcg(p.part_lse + it * p.rows + r);
                    x[cc] = __ldcg(reinterpret_cast<const float2*>(p.part_o + (it * p.rows + r) * kD + d));
                } else {
                    lse[cc] = -INFINITY;
                    x[cc] = make_float2(0.f, 0.f);
                }
            }
            const float mx = fmaxf(fmaxf(mrun, fmaxf(lse[0], lse[1])), fmaxf(lse[2], lse[3]));
            if (mx == -INFINITY) continue;
            const float sc = mrun == -INFINITY ? 0.f : fast_exp2(mrun - mx);
            den *= sc;
            acc0 *= sc;
            acc1 *= sc;
#pragma unroll
            for (int cc = 0; cc < 4; ++cc) {
                const float w = lse[cc] == -INFINITY ? 0.f : fast_exp2(lse[cc] - mx);
                den += w;
                acc0 = fmaf(w, x[cc].x, acc0);
                acc1 = fmaf(w, x[cc].y, acc1);
            }
            mrun = mx;
        }
        const float inv = den > 0.f ? 1.f / den : 0.f;
        const int j = r / p.group, gq = r - j * p.group;
        *reinterpret_cast<uint32_t*>(p.out + ((int64_t(hd.b) * p.lq + j) * p.hq + hd.h * p.group + gq) * kD +
                                     d) = pack2<BF16>(acc0 * inv, acc1 * inv);
    }
}

}  // namespace pa
}  // namespace b200
