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
// whose records are neighbours in a page (160 bytes, five whole sectors).  A block takes
// a run of tokens, looks their slots up once and deals the (token pair, row) tasks to its warps.
#include "kv_q4.cuh"

namespace b200 {
namespace q4 {
namespace {

constexpr int kWarps = 8;
constexpr int kMaxTokens = 32;  // tokens of one block

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

__device__ __forceinline__ int64_t record_offset(const Cache& c, int64_t slot, int h) {
    const uint32_t blk = uint32_t(slot) / uint32_t(c.block_size);
    return ((int64_t(blk) * c.hkv + h) * c.block_size + (uint32_t(slot) - blk * c.block_size)) * kRecord;
}

// Runs f(token of the block, row of the token, half-warp lane) over all rows of `count` tokens;
// both halves of a warp call it together (the token may be past the end: the caller masks it).
template <typename F>
__device__ __forceinline__ void for_rows(int count, int rows, F f) {
    const int lane = threadIdx.x & 31;
    const int tasks = ((count + 1) / 2) * rows;
    for (int i = threadIdx.x >> 5; i < tasks; i += kWarps) {
        const int pair = i / rows;
        f(2 * pair + (lane >> 4), i - pair * rows, lane & 15);
    }
}

template <bool BF16, bool VEC>
__global__ void __launch_bounds__(kWarps * 32)
    store_kernel(const Rows rows, const Cache cache, const int32_t* __restrict__ slots, int32_t n, int32_t tokens) {
    __shared__ int32_t s_slot[kMaxTokens];
    const int64_t t0 = int64_t(blockIdx.x) * tokens;
    const int count = int(min(int64_t(tokens), n - t0));
    if (threadIdx.x < kMaxTokens) {
        const int32_t s = threadIdx.x < count ? slots[t0 + threadIdx.x] : -1;
        s_slot[threadIdx.x] = s < cache.num_slots ? s : -1;
    }
    __syncthreads();
    for_rows(count, 2 * cache.hkv, [&](int t, int r, int l) {
        const bool is_v = r >= cache.hkv;
        const int h = is_v ? r - cache.hkv : r;
        const int32_t slot = t < kMaxTokens ? s_slot[t] : -1;
        uint32_t x[4] = {0, 0, 0, 0};
        if (slot >= 0) {
            const char* src = (is_v ? rows.v + (t0 + t) * rows.v_stride : rows.k + (t0 + t) * rows.k_stride) +
                              (h * kD + 8 * l) * 2;
            if constexpr (VEC) {
                const uint4 v = __ldg(reinterpret_cast<const uint4*>(src));
                x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
            } else {
                const uint16_t* e = reinterpret_cast<const uint16_t*>(src);
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = uint32_t(e[2 * i]) | (uint32_t(e[2 * i + 1]) << 16);
            }
        }
        uint32_t params;
        const uint32_t word = quantise8<BF16>(x, params);
        if (slot >= 0) {
            char* rec = (is_v ? cache.v : cache.k) + record_offset(cache, slot, h);
            *reinterpret_cast<uint32_t*>(rec + 4 * l) = word;
            if ((l & 3) == 0) *reinterpret_cast<uint32_t*>(rec + kParams + l) = params;
        }
    });
}

// Slots of a block's tokens for the readers: kZero for rows that read as zeros, kSkip for rows
// that are left as they were.
constexpr int32_t kZero = -1, kSkip = -2;

template <bool BF16, bool VEC>
__device__ __forceinline__ void read_rows(const Rows& rows, const Cache& cache, const int32_t* s_slot, int64_t t0,
                                          int count) {
    for_rows(count, 2 * cache.hkv, [&](int t, int r, int l) {
        const bool is_v = r >= cache.hkv;
        const int h = is_v ? r - cache.hkv : r;
        const int32_t slot = t < count ? s_slot[t] : kSkip;
        if (slot == kSkip) return;
        uint4 y = make_uint4(0, 0, 0, 0);
        if (slot >= 0) {
            const char* rec = (is_v ? cache.v : cache.k) + record_offset(cache, slot, h);
            y = dequantise8<BF16>(*reinterpret_cast<const uint32_t*>(rec + 4 * l),
                                  *reinterpret_cast<const uint32_t*>(rec + kParams + (l & ~3)));
        }
        char* dst = (is_v ? rows.v + (t0 + t) * rows.v_stride : rows.k + (t0 + t) * rows.k_stride) +
                    (h * kD + 8 * l) * 2;
        if constexpr (VEC) {
            *reinterpret_cast<uint4*>(dst) = y;
        } else {
            const uint32_t w[4] = {y.x, y.y, y.z, y.w};
            uint16_t* e = reinterpret_cast<uint16_t*>(dst);
#pragma unroll
            for (int i = 0; i < 4; ++i) e[2 * i] = uint16_t(w[i]), e[2 * i + 1] = uint16_t(w[i] >> 16);
        }
    });
}

template <bool BF16, bool VEC>
__global__ void __launch_bounds__(kWarps * 32)
    load_kernel(const Rows rows, const Cache cache, const int32_t* __restrict__ slots, int32_t n, int32_t tokens) {
    __shared__ int32_t s_slot[kMaxTokens];
    const int64_t t0 = int64_t(blockIdx.x) * tokens;
    const int count = int(min(int64_t(tokens), n - t0));
    if (threadIdx.x < count) {
        const int32_t s = slots[t0 + threadIdx.x];
        s_slot[threadIdx.x] = s >= 0 && s < cache.num_slots ? s : kZero;
    }
    __syncthreads();
    read_rows<BF16, VEC>(rows, cache, s_slot, t0, count);
}

template <bool BF16, bool VEC>
__global__ void __launch_bounds__(kWarps * 32)
    gather_kernel(const Rows rows, const Cache cache, const int32_t* __restrict__ cu, const int32_t* __restrict__ tables,
                  int64_t bt_stride, int32_t bt_width, int32_t num_seqs, int32_t n, int32_t tokens) {
    __shared__ int32_t s_slot[kMaxTokens];
    const int64_t t0 = int64_t(blockIdx.x) * tokens;
    const int count = int(min(int64_t(tokens), n - t0));
    if (threadIdx.x < count) {
        const int32_t t = int32_t(t0) + threadIdx.x;
        int32_t slot = kSkip;
        if (t >= cu[0] && t < cu[num_seqs]) {  // else: a row of no sequence
            int lo = 0, hi = num_seqs;         // the last sequence that starts at or before t
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (cu[mid] <= t) lo = mid; else hi = mid;
            }
            const uint32_t pos = uint32_t(t - cu[lo]), page = pos / uint32_t(cache.block_size);
            slot = kZero;
            if (page < uint32_t(bt_width)) {
                const int32_t blk = tables[lo * bt_stride + page];
                if (blk >= 0 && int64_t(blk) * cache.block_size < cache.num_slots)
                    slot = blk * cache.block_size + int32_t(pos - page * cache.block_size);
            }
        }
        s_slot[threadIdx.x] = slot;
    }
    __syncthreads();
    read_rows<BF16, VEC>(rows, cache, s_slot, t0, count);
}

// Tokens per block: at least two blocks per SM while there are tokens to spare (a small call is
// latency, spread it), at most kMaxTokens (a large one looks its slots up in bulk).
int tokens_per_block(int32_t n) {
    const int64_t blocks = 4 * int64_t(device_sm_count());
    int t = 2;
    while (t < kMaxTokens && n > blocks * t) t *= 2;
    return t;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int32_t check_common(const char* what, const void* k_rows, int64_t k_stride, const void* v_rows, int64_t v_stride,
                     const void* k_cache, const void* v_cache, int32_t num_tokens, int32_t num_kv_heads,
                     int32_t head_dim, int32_t num_blocks, int32_t block_size, int32_t dtype) {
    B200_REQUIRE(k_rows && v_rows && k_cache && v_cache, "%s: null pointer", what);
    B200_REQUIRE(num_kv_heads > 0 && num_kv_heads <= 32768, "%s: num_kv_heads %d", what, num_kv_heads);
    if (head_dim != kD) return fail(B200_ERR_UNSUPPORTED, "%s: head_dim %d (only 128)", what, head_dim);
    if (dtype != B200_BF16 && dtype != B200_F16)
        return fail(B200_ERR_UNSUPPORTED, "%s: dtype %d (bf16 or fp16 only)", what, dtype);
    B200_REQUIRE(num_blocks > 0 && block_size > 0 && int64_t(num_blocks) * block_size < (int64_t(1) << 31),
                 "%s: %d blocks of %d tokens", what, num_blocks, block_size);
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

// Launches KERNEL<BF16, VEC> for the call's type and alignment.
#define B200_Q4_LAUNCH(KERNEL, grid, stream, ...)                                                     \
    do {                                                                                              \
        const bool vec_ = vector_rows(rows);                                                          \
        if (dtype == B200_BF16) {                                                                     \
            if (vec_) KERNEL<true, true><<<grid, kWarps * 32, 0, stream>>>(__VA_ARGS__);              \
            else KERNEL<true, false><<<grid, kWarps * 32, 0, stream>>>(__VA_ARGS__);                  \
        } else {                                                                                      \
            if (vec_) KERNEL<false, true><<<grid, kWarps * 32, 0, stream>>>(__VA_ARGS__);             \
            else KERNEL<false, false><<<grid, kWarps * 32, 0, stream>>>(__VA_ARGS__);                 \
        }                                                                                             \
        B200_CUDA_TRY(cudaGetLastError());                                                            \
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
    const int tokens = tokens_per_block(num_tokens);
    const dim3 grid((unsigned(num_tokens) + tokens - 1) / tokens);
    B200_Q4_LAUNCH(store_kernel, grid, static_cast<cudaStream_t>(stream), rows, cache, slot_mapping, num_tokens, tokens);
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
    const int tokens = tokens_per_block(num_tokens);
    const dim3 grid((unsigned(num_tokens) + tokens - 1) / tokens);
    B200_Q4_LAUNCH(load_kernel, grid, static_cast<cudaStream_t>(stream), rows, cache, slot_mapping, num_tokens, tokens);
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
    const int tokens = tokens_per_block(total_tokens);
    const dim3 grid((unsigned(total_tokens) + tokens - 1) / tokens);
    B200_Q4_LAUNCH(gather_kernel, grid, static_cast<cudaStream_t>(stream), rows, cache, cu_seqlens, block_tables,
                   block_table_stride, block_table_width, num_seqs, total_tokens, tokens);
    return B200_OK;
}
