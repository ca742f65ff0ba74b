// Writing a 4-bit KV cache and reading it back.
//
//   store   quantises the key and value rows of new tokens into the records of their slots
//           (the 4-bit counterpart of store_kvcache, nanovllm/layers/attention.py:10-40);
//   load    reads the records of a list of slots back as rows of the model's type;
//   gather  reads whole sequences back through their block tables as packed rows, the layout
//           the varlen prefill takes (attention.py:64-70 reads such sequences from the cache).
//
// All three are bound by memory: 512 bytes of rows and 160 bytes of records per (token, kv
// head).  A half-warp owns a row (16 bytes, eight dimensions, per lane), so that the four
// lanes of a quad hold one group: two shuffles find its extremes and every lane ends with one
// whole word of codes.  The two halves of a warp take the same head of two consecutive tokens,
// whose records are neighbours in a page (160 bytes, five whole sectors).  A block takes a run
// of tokens and looks up once where their records lie; each of its warps takes rows (a head's
// keys or values) and walks the token pairs, kFlight of them in flight.
#include <algorithm>

#include "kv_q4.cuh"

namespace b200 {
namespace q4 {
namespace {

constexpr int kWarps = 8;
constexpr int kMaxTokens = 32;  // of one block
// Resident blocks per SM (launch bounds) and tokens of a block where many waves run: see shape_of.
constexpr int kStoreBlocks = 4, kStoreTokens = 24;
constexpr int kReadBlocks = 5, kReadTokens = 16;

struct Rows {
    char* k;  // key rows (read by store, written by load and gather)
    char* v;
    int64_t k_stride, v_stride;  // bytes between tokens
};

struct Cache {
    char* k;
    char* v;
    int32_t hkv, block_size;
    int64_t num_slots;
};

// Index of head 0's record of a slot (heads are block_size records apart).  All records of a cache
// have 32-bit indices, which leaves one multiply-add per address.
__device__ __forceinline__ uint32_t record_of(const Cache& c, int32_t slot) {
    const uint32_t blk = uint32_t(slot) / uint32_t(c.block_size);
    return blk * uint32_t(c.hkv) * uint32_t(c.block_size) + (uint32_t(slot) - blk * c.block_size);
}

// Tokens without a record: rows that read as zeros, rows that are left alone.
constexpr uint32_t kZero = 0xffffffffu, kSkip = 0xfffffffeu;

// Deals the rows of `count` tokens to the block's warps and calls, kFlight pairs at a time, LOAD and then
// USE for each: (u, index of the token's record, the head's records, the lane's 16 bytes of the row).
// Both halves of a warp run together; past the last pair the index is kSkip.
template <int kFlight, typename LOAD, typename USE>
__device__ __forceinline__ void for_rows(const Rows& rows, const Cache& cache, const uint32_t* s_rec, int64_t t0, int count,
                                         LOAD load, USE use) {
    const int half = (threadIdx.x >> 4) & 1, l = threadIdx.x & 15, pairs = (count + 1) >> 1;
#pragma unroll 1  // a block comes by once or twice: more code is more to fetch
    for (int r = blockIdx.y * kWarps + (threadIdx.x >> 5); r < 2 * cache.hkv; r += gridDim.y * kWarps) {
        const bool v = r >= cache.hkv;
        const int h = v ? r - cache.hkv : r;
        const int64_t stride = v ? rows.v_stride : rows.k_stride;
        char* row = (v ? rows.v : rows.k) + (t0 + half) * stride + h * (kD * 2) + 16 * l;
        char* records = (v ? cache.v : cache.k) + int64_t(h) * cache.block_size * kRecord;
#pragma unroll 1
        for (int p0 = 0; p0 < pairs; p0 += kFlight) {
            uint32_t rec[kFlight];
#pragma unroll
            for (int u = 0; u < kFlight; ++u) {
                rec[u] = p0 + u < pairs ? s_rec[2 * (p0 + u) + half] : kSkip;
                load(u, rec[u], records, row + u * 2 * stride);
            }
#pragma unroll
            for (int u = 0; u < kFlight; ++u) use(u, rec[u], records, row + u * 2 * stride);
            row += kFlight * 2 * stride;
        }
    }
}

template <bool BF16, bool VEC, int kFlight>
__global__ void __launch_bounds__(kWarps * 32, kStoreBlocks)
    store_kernel(const Rows rows, const Cache cache, const int32_t* __restrict__ slots, int32_t n, int32_t tokens) {
    __shared__ uint32_t s_rec[kMaxTokens];
    const int64_t t0 = int64_t(blockIdx.x) * tokens;
    const int count = int(min(int64_t(tokens), n - t0));
    if (threadIdx.x < kMaxTokens) {
        const int32_t s = threadIdx.x < count ? slots[t0 + threadIdx.x] : -1;
        s_rec[threadIdx.x] = s >= 0 && s < cache.num_slots ? record_of(cache, s) : kSkip;
    }
    __syncthreads();
    const int l = threadIdx.x & 15;
    uint32_t x[kFlight][4];
    for_rows<kFlight>(
        rows, cache, s_rec, t0, count,
        [&](int u, uint32_t rec, char*, char* row) {
            x[u][0] = x[u][1] = x[u][2] = x[u][3] = 0;
            if (rec >= kSkip) return;
            if constexpr (VEC) {
                const uint4 w = __ldg(reinterpret_cast<const uint4*>(row));
                x[u][0] = w.x, x[u][1] = w.y, x[u][2] = w.z, x[u][3] = w.w;
            } else {
                const uint16_t* e = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
                for (int i = 0; i < 4; ++i) x[u][i] = uint32_t(e[2 * i]) | (uint32_t(e[2 * i + 1]) << 16);
            }
        },
        [&](int u, uint32_t rec, char* records, char*) {
            uint32_t params;
            const uint32_t word = quantise8<BF16>(x[u], params);
            if (rec >= kSkip) return;
            *reinterpret_cast<uint32_t*>(records + int64_t(rec) * kRecord + 4 * l) = word;
            if ((l & 3) == 0) *reinterpret_cast<uint32_t*>(records + int64_t(rec) * kRecord + kParams + l) = params;
        });
}

template <bool BF16, bool VEC, int kFlight>
__device__ __forceinline__ void read_rows(const Rows& rows, const Cache& cache, const uint32_t* s_rec, int64_t t0,
                                          int count) {
    const int l = threadIdx.x & 15;
    uint32_t word[kFlight], params[kFlight];
    for_rows<kFlight>(
        rows, cache, s_rec, t0, count,
        [&](int u, uint32_t rec, char* records, char*) {
            word[u] = params[u] = 0;
            if (rec >= kSkip) return;
            word[u] = __ldg(reinterpret_cast<const uint32_t*>(records + int64_t(rec) * kRecord + 4 * l));
            params[u] = __ldg(reinterpret_cast<const uint32_t*>(records + int64_t(rec) * kRecord + kParams + (l & ~3)));
        },
        [&](int u, uint32_t rec, char*, char* row) {
            if (rec == kSkip) return;
            const uint4 y = dequantise8<BF16>(word[u], params[u]);  // no record: zeros
            if constexpr (VEC) {
                *reinterpret_cast<uint4*>(row) = y;
            } else {
                const uint32_t w[4] = {y.x, y.y, y.z, y.w};
                uint16_t* e = reinterpret_cast<uint16_t*>(row);
#pragma unroll
                for (int i = 0; i < 4; ++i) e[2 * i] = uint16_t(w[i]), e[2 * i + 1] = uint16_t(w[i] >> 16);
            }
        });
}

template <bool BF16, bool VEC, int kFlight>
__global__ void __launch_bounds__(kWarps * 32, kReadBlocks)
    load_kernel(const Rows rows, const Cache cache, const int32_t* __restrict__ slots, int32_t n, int32_t tokens) {
    __shared__ uint32_t s_rec[kMaxTokens];
    const int64_t t0 = int64_t(blockIdx.x) * tokens;
    const int count = int(min(int64_t(tokens), n - t0));
    if (threadIdx.x < kMaxTokens) {
        uint32_t rec = kSkip;
        if (threadIdx.x < count) {
            const int32_t s = slots[t0 + threadIdx.x];
            rec = s >= 0 && s < cache.num_slots ? record_of(cache, s) : kZero;
        }
        s_rec[threadIdx.x] = rec;
    }
    __syncthreads();
    read_rows<BF16, VEC, kFlight>(rows, cache, s_rec, t0, count);
}

template <bool BF16, bool VEC, int kFlight>
__global__ void __launch_bounds__(kWarps * 32, kReadBlocks)
    gather_kernel(const Rows rows, const Cache cache, const int32_t* __restrict__ cu, const int32_t* __restrict__ tables,
                  int64_t bt_stride, int32_t bt_width, int32_t num_seqs, int32_t n, int32_t tokens) {
    __shared__ uint32_t s_rec[kMaxTokens];
    const int64_t t0 = int64_t(blockIdx.x) * tokens;
    const int count = int(min(int64_t(tokens), n - t0));
    if (threadIdx.x < kMaxTokens) {
        const int32_t t = int32_t(t0) + threadIdx.x;
        uint32_t rec = kSkip;
        if (threadIdx.x < count && t >= cu[0] && t < cu[num_seqs]) {  // else: a row of no sequence
            int lo = 0, hi = num_seqs;                               // the last sequence that starts at or before t
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (cu[mid] <= t) lo = mid; else hi = mid;
            }
            const uint32_t pos = uint32_t(t - cu[lo]), page = pos / uint32_t(cache.block_size);
            rec = kZero;
            if (page < uint32_t(bt_width)) {
                const int32_t blk = tables[lo * bt_stride + page];
                if (blk >= 0 && int64_t(blk) * cache.block_size < cache.num_slots)
                    rec = record_of(cache, blk * cache.block_size + int32_t(pos - page * cache.block_size));
            }
        }
        s_rec[threadIdx.x] = rec;
    }
    __syncthreads();
    read_rows<BF16, VEC, kFlight>(rows, cache, s_rec, t0, count);
}

// Launch shape.  Up to two tokens per resident block: latency, a pair of tokens per block and a row per
// warp (8 tokens x 8 heads, store and load in a graph: 3.6 us against 5.4 with four pairs in flight).
// More: four pairs per warp in flight, at least three of them full (2500 tokens, store and load: 8.7 us
// against 9.5 with two; 1500: 7.2, with four 7.7); one wave of resident blocks while they can hold it
// (16,384 tokens: 37 us against 38.3 in two waves), else whole waves of shorter blocks (gather of 68.6k tokens:
// 53.2 us with up to 16 tokens, 55.2 with 24; store and load of 40,000: 86.4 us with 24 tokens in the store's, 89.0
// with 16).  Reading wants the fifth block of 48 registers (gather of four sequences of 26k: 104.8 us against
// 111.7), storing loses by it (16,384 tokens: 39.5 us).
struct Shape {
    int tokens;
    dim3 grid;
    bool small;
};

Shape shape_of(int32_t n, int32_t hkv, int per_sm, int wave_tokens) {
    const int64_t blocks = int64_t(per_sm) * device_sm_count();
    Shape s;
    s.small = n <= 2 * blocks;
    const int64_t waves = n <= kMaxTokens * blocks ? 1 : (n + wave_tokens * blocks - 1) / (wave_tokens * blocks);
    s.tokens = s.small ? 2 : std::max(6, int((n + waves * blocks - 1) / (waves * blocks) + 1) & ~1);
    s.grid = dim3((unsigned(n) + s.tokens - 1) / s.tokens, s.small ? (2 * hkv + kWarps - 1) / kWarps : 1);
    return s;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int32_t check_common(const char* what, const void* k_rows, int64_t k_stride, const void* v_rows, int64_t v_stride,
                     const void* k_cache, const void* v_cache, int32_t num_tokens, int32_t num_kv_heads,
                     int32_t head_dim, int32_t num_blocks, int32_t block_size, int32_t dtype) {
    B200_REQUIRE(k_rows && v_rows && k_cache && v_cache, "%s: null pointer", what);
    B200_REQUIRE(num_kv_heads > 0 && num_kv_heads <= 65535, "%s: num_kv_heads %d", what, num_kv_heads);
    if (head_dim != kD) return fail(B200_ERR_UNSUPPORTED, "%s: head_dim %d (only 128)", what, head_dim);
    if (dtype != B200_BF16 && dtype != B200_F16)
        return fail(B200_ERR_UNSUPPORTED, "%s: dtype %d (bf16 or fp16 only)", what, dtype);
    B200_REQUIRE(num_blocks > 0 && block_size > 0 && int64_t(num_blocks) * block_size < (int64_t(1) << 31),
                 "%s: %d blocks of %d tokens", what, num_blocks, block_size);
    if (int64_t(num_blocks) * block_size > int64_t(kSkip) / num_kv_heads)
        return fail(B200_ERR_UNSUPPORTED, "%s: %d blocks of %d tokens and %d heads: more than 2^32 records", what,
                    num_blocks, block_size, num_kv_heads);
    const int64_t row = int64_t(num_kv_heads) * kD;
    B200_REQUIRE(num_tokens <= 1 || (k_stride >= row && v_stride >= row), "%s: token stride (%lld, %lld) below Hkv*D = %lld",
                 what, (long long)k_stride, (long long)v_stride, (long long)row);
    B200_REQUIRE(aligned16(k_cache) && aligned16(v_cache), "%s: caches must be 16-byte aligned", what);
    B200_REQUIRE((reinterpret_cast<uintptr_t>(k_rows) & 1) == 0 && (reinterpret_cast<uintptr_t>(v_rows) & 1) == 0,
                 "%s: rows must be 2-byte aligned", what);
    return B200_OK;
}

bool vector_rows(const Rows& r) {
    return aligned16(r.k) && aligned16(r.v) && r.k_stride % 16 == 0 && r.v_stride % 16 == 0;
}

// Launches KERNEL for the call's type, alignment and shape.
#define B200_Q4_CASE(KERNEL, BF16, VEC, ...)                                                  \
    do {                                                                                      \
        if (shape.small) KERNEL<BF16, VEC, 1><<<shape.grid, kWarps * 32, 0, st>>>(__VA_ARGS__); \
        else KERNEL<BF16, VEC, 4><<<shape.grid, kWarps * 32, 0, st>>>(__VA_ARGS__);           \
    } while (0)
#define B200_Q4_LAUNCH(KERNEL, PER_SM, n, ...)                                           \
    do {                                                                         \
        const Shape shape = shape_of(n, num_kv_heads, PER_SM##Blocks, PER_SM##Tokens);                           \
        cudaStream_t st = static_cast<cudaStream_t>(stream);                     \
        const bool vec = vector_rows(rows);                                      \
        if (dtype == B200_BF16 && vec) B200_Q4_CASE(KERNEL, true, true, __VA_ARGS__, shape.tokens);  \
        else if (dtype == B200_BF16) B200_Q4_CASE(KERNEL, true, false, __VA_ARGS__, shape.tokens);   \
        else if (vec) B200_Q4_CASE(KERNEL, false, true, __VA_ARGS__, shape.tokens);                  \
        else B200_Q4_CASE(KERNEL, false, false, __VA_ARGS__, shape.tokens);                          \
        B200_CUDA_TRY(cudaGetLastError());                                       \
    } while (0)

}  // namespace
}  // namespace q4
}  // namespace b200

extern "C" int32_t b200_store_kvcache_q4(const void* key, int64_t key_stride, const void* value, int64_t value_stride,
                                         void* k_cache, void* v_cache, const int32_t* slot_mapping,
                                         int32_t num_tokens, int32_t num_kv_heads, int32_t head_dim,
                                         int32_t num_blocks, int32_t block_size, int32_t dtype, void* stream) {
    using namespace b200;
    using namespace b200::q4;
    clear_error();
    B200_REQUIRE(num_tokens >= 0, "store_kvcache_q4: num_tokens %d < 0", num_tokens);
    if (num_tokens == 0) return B200_OK;
    B200_REQUIRE(slot_mapping, "store_kvcache_q4: null pointer");
    const int32_t rc = check_common("store_kvcache_q4", key, key_stride, value, value_stride, k_cache, v_cache,
                                    num_tokens, num_kv_heads, head_dim, num_blocks, block_size, dtype);
    if (rc) return rc;
    const Rows rows{static_cast<char*>(const_cast<void*>(key)), static_cast<char*>(const_cast<void*>(value)),
                    key_stride * 2, value_stride * 2};
    const Cache cache{static_cast<char*>(k_cache), static_cast<char*>(v_cache), num_kv_heads, block_size,
                      int64_t(num_blocks) * block_size};
    B200_Q4_LAUNCH(store_kernel, kStore, num_tokens, rows, cache, slot_mapping, num_tokens);
    return B200_OK;
}

extern "C" int32_t b200_load_kvcache_q4(void* key, int64_t key_stride, void* value, int64_t value_stride,
                                        const void* k_cache, const void* v_cache, const int32_t* slot_mapping,
                                        int32_t num_tokens, int32_t num_kv_heads, int32_t head_dim,
                                        int32_t num_blocks, int32_t block_size, int32_t dtype, void* stream) {
    using namespace b200;
    using namespace b200::q4;
    clear_error();
    B200_REQUIRE(num_tokens >= 0, "load_kvcache_q4: num_tokens %d < 0", num_tokens);
    if (num_tokens == 0) return B200_OK;
    B200_REQUIRE(slot_mapping, "load_kvcache_q4: null pointer");
    const int32_t rc = check_common("load_kvcache_q4", key, key_stride, value, value_stride, k_cache, v_cache,
                                    num_tokens, num_kv_heads, head_dim, num_blocks, block_size, dtype);
    if (rc) return rc;
    const Rows rows{static_cast<char*>(key), static_cast<char*>(value), key_stride * 2, value_stride * 2};
    const Cache cache{static_cast<char*>(const_cast<void*>(k_cache)), static_cast<char*>(const_cast<void*>(v_cache)),
                      num_kv_heads, block_size, int64_t(num_blocks) * block_size};
    B200_Q4_LAUNCH(load_kernel, kRead, num_tokens, rows, cache, slot_mapping, num_tokens);
    return B200_OK;
}

extern "C" int32_t b200_gather_kvcache_q4(void* key, int64_t key_stride, void* value, int64_t value_stride,
                                          const void* k_cache, const void* v_cache, const int32_t* cu_seqlens,
                                          const int32_t* block_tables, int64_t block_table_stride,
                                          int32_t block_table_width, int32_t num_seqs, int32_t total_tokens, int32_t num_kv_heads, int32_t head_dim,
                                          int32_t num_blocks, int32_t block_size, int32_t dtype, void* stream) {
    using namespace b200;
    using namespace b200::q4;
    clear_error();
    B200_REQUIRE(total_tokens >= 0 && num_seqs >= 0, "gather_kvcache_q4: %d sequences, %d tokens", num_seqs, total_tokens);
    if (total_tokens == 0 || num_seqs == 0) return B200_OK;
    B200_REQUIRE(cu_seqlens && block_tables, "gather_kvcache_q4: null pointer");
    B200_REQUIRE(block_table_width > 0 && block_table_stride >= 0,
                 "gather_kvcache_q4: block table of %d entries, stride %lld", block_table_width,
                 (long long)block_table_stride);
    const int32_t rc = check_common("gather_kvcache_q4", key, key_stride, value, value_stride, k_cache, v_cache,
                                    total_tokens, num_kv_heads, head_dim, num_blocks, block_size, dtype);
    if (rc) return rc;
    const Rows rows{static_cast<char*>(key), static_cast<char*>(value), key_stride * 2, value_stride * 2};
    const Cache cache{static_cast<char*>(const_cast<void*>(k_cache)), static_cast<char*>(const_cast<void*>(v_cache)),
                      num_kv_heads, block_size, int64_t(num_blocks) * block_size};
    B200_Q4_LAUNCH(gather_kernel, kRead, total_tokens, rows, cache, cu_seqlens, block_tables, block_table_stride,
                   block_table_width, num_seqs, total_tokens);
    return B200_OK;
}
