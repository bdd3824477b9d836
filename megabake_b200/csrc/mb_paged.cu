// Operators around a paged key-value cache: pages and slots for new tokens (mb_paged_reserve), keys and
// values into their slots (mb_paged_append), attention of one new token a request (mb_paged_attention) and of
// several (mb_paged_prefill).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <initializer_list>

#include "mb_device.cuh"
#include "mb_kernels.h"
#include "mb_paged.cuh"

namespace mb {
namespace paged {

// ---------------------------------------------------------------------------------------
// Pages and slots from request lengths
//
// Three exclusive sums over the requests decide everything: pages given back by the rows behind r (where r's pages
// go on the stack), tokens and pages wanted by the rows up to r (whether r is granted), tokens and pages granted
// before r (its places, and which entries of the stack are its pages).  A thread sums a run of neighbouring rows, the
// block scans the threads; what a row looks up afterwards lies in shared memory.
//
// Latency bounds it: one trip to L2 after the other (lengths, pages given back, pages granted, slots), and with many
// tokens 20 bytes for each of their places.  A thread-block cluster shares the rows and places, and every block of it
// works the sums out for itself: its barrier is all that tables which are read and updated in one launch need.
// ---------------------------------------------------------------------------------------
//
// A few requests: one block of four warps, whose barriers and sums are the shortest (32 requests, reserved and taken back:
// 9.6 us with 128 threads, 10.4 with 512).  Otherwise eight blocks of 512 (of 1,024, 256 requests: 34.7 us, not 32.1).
constexpr int kReserveCluster = 8;

struct ReserveArgs {
    int requests, width, pages, page_shift, max_tokens;
    const int* counts;
    int *lengths, *table, *stack, *free_count, *offsets, *rows, *granted;
    long long *slots, *positions;
};

struct Pair {
    long long a, b;
};

__device__ __forceinline__ Pair inclusive_sums(Pair v, int lane) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long a = __shfl_up_sync(0xffffffffu, v.a, d);
        const long long b = __shfl_up_sync(0xffffffffu, v.b, d);
        if (lane >= d) {
            v.a += a;
            v.b += b;
        }
    }
    return v;
}

// Exclusive sums over the threads of the block, and the totals.  Every thread calls it.
template <int kThreads>
__device__ __forceinline__ Pair exclusive_sums(Pair v, Pair* warp_sums, Pair& total) {
    constexpr int kWarps = kThreads / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Pair mine = inclusive_sums(v, lane);
    __syncthreads();  // the sums of a call before have been read
    if (lane == 31) warp_sums[warp] = mine;
    __syncthreads();
    const Pair warps = inclusive_sums(lane < kWarps ? warp_sums[lane] : Pair{0, 0}, lane);
    total = {__shfl_sync(0xffffffffu, warps.a, kWarps - 1), __shfl_sync(0xffffffffu, warps.b, kWarps - 1)};
    const Pair before = {__shfl_sync(0xffffffffu, warps.a, (warp + 31) & 31),
                         __shfl_sync(0xffffffffu, warps.b, (warp + 31) & 31)};
    return {(warp > 0 ? before.a : 0) + mine.a - v.a, (warp > 0 ? before.b : 0) + mine.b - v.b};
}

// Everything the cluster wrote before is seen by all of it afterwards; what lies in L1 from before is not used again.
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <int kThreads>
__global__ void __launch_bounds__(kThreads) reserve_kernel(const ReserveArgs p) {
    extern __shared__ int rows_smem[];
    const int R = p.requests, page = 1 << p.page_shift;
    int* held_tokens = rows_smem;           // [R] tokens at first
    int* kept_tokens = rows_smem + R;       // [R] that stay before any are granted
    int* first_page = rows_smem + 2 * R;    // [R] pages given back by later rows, then pages granted to earlier ones
    int* offset = rows_smem + 3 * R;        // [R + 1]
    __shared__ Pair warp_sums[kThreads / 32];
    // gridDim.x is the cluster
    const int tid = threadIdx.x, rank = blockIdx.x, everyone = gridDim.x * kThreads, me = rank * kThreads + tid;
    const int per_thread = (R + kThreads - 1) / kThreads;
    const int r0 = min(tid * per_thread, R), r1 = min(r0 + per_thread, R);
    const int capacity = p.width << p.page_shift;
    auto pages_of = [&](long long tokens) { return static_cast<int>((tokens + page - 1) >> p.page_shift); };

    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int free_before = *p.free_count;
    Pair back = {0, 0}, wanted = {0, 0}, total;
    for (int r = r0; r < r1; ++r) {
        const int count = p.counts[r], held = min(max(p.lengths[r], 0), capacity);
        const int kept = count < 0 ? static_cast<int>(max(static_cast<long long>(held) + count, 0ll)) : held;
        held_tokens[r] = held;
        kept_tokens[r] = kept;
        offset[r] = 0;
        back.a += pages_of(held) - pages_of(kept);
        const long long after = static_cast<long long>(kept) + count;
        if (count > 0 && after <= capacity) {
            offset[r] = count;   // what it wants
            wanted.a += count;
            wanted.b += pages_of(after) - pages_of(kept);
        }
    }
    // what is given back
    Pair before = exclusive_sums<kThreads>(back, warp_sums, total);
    const long long given = total.a, available = free_before + given;
    long long behind = total.a - before.a;
    for (int r = r0; r < r1; ++r) {
        behind -= pages_of(held_tokens[r]) - pages_of(kept_tokens[r]);
        first_page[r] = static_cast<int>(behind);
    }
    if (given > 0) {
        __syncthreads();
        for (long long k = me; k < given; k += everyone) {   // a page a thread: the k-th that goes on the stack
            int low = 0, high = R - 1;                       // the first row that gives no more than k pages behind it
            while (low < high) {
                const int middle = (low + high) >> 1;
                if (first_page[middle] <= k)
                    high = middle;
                else
                    low = middle + 1;
            }
            const long long j = pages_of(held_tokens[low]) - 1 - (k - first_page[low]), at = free_before + k;
            int* entry = p.table + static_cast<size_t>(low) * p.width + j;
            if (at >= 0 && at < p.pages) p.stack[at] = *entry;
            *entry = -1;
        }
    }

    // who is granted what he wants
    before = exclusive_sums<kThreads>(wanted, warp_sums, total);
    Pair got = {0, 0};
    for (int r = r0; r < r1; ++r) {
        const int count = offset[r];
        if (count > 0) {
            const int need = pages_of(static_cast<long long>(kept_tokens[r]) + count) - pages_of(kept_tokens[r]);
            before.a += count;
            before.b += need;
            if (before.a <= p.max_tokens && (need == 0 || before.b <= available)) {
                got.a += count;
                got.b += need;
            } else {
                offset[r] = 0;
            }
        }
    }
    before = exclusive_sums<kThreads>(got, warp_sums, total);
    for (int r = r0; r < r1; ++r) {
        const int count = offset[r];
        offset[r] = static_cast<int>(before.a);
        first_page[r] = static_cast<int>(before.b);
        before.a += count;
        before.b += pages_of(static_cast<long long>(kept_tokens[r]) + count) - pages_of(kept_tokens[r]);
    }
    if (tid == 0) offset[R] = static_cast<int>(total.a);
    cluster_barrier();  // lengths, counts and the free count have been read; the pages given back are on the stack
    for (long long k = me; k < total.b; k += everyone) {   // a page a thread: the k-th that is granted
        int low = 0, high = R;                             // first_page[low] <= k, the last such row
        while (high - low > 1) {
            const int middle = (low + high) >> 1;
            if (first_page[middle] <= k)
                low = middle;
            else
                high = middle;
        }
        const long long at = available - 1 - k;
        p.table[static_cast<size_t>(low) * p.width + pages_of(kept_tokens[low]) + (k - first_page[low])] =
            at >= 0 && at < p.pages ? __ldcg(p.stack + at) : -1;
    }
    if (rank == 0) {
        for (int r = tid; r < R; r += kThreads) {
            const int count = offset[r + 1] - offset[r];
            p.granted[r] = count > 0 ? count : kept_tokens[r] - held_tokens[r];
            p.lengths[r] = kept_tokens[r] + count;
            p.offsets[r] = offset[r];
        }
        if (tid == 0) {
            p.offsets[R] = offset[R];
            *p.free_count = static_cast<int>(available - total.b);
        }
    }
    if (total.b > 0) cluster_barrier();  // the table is complete
    // four places a thread: one search, and as a rule one entry of the table
    for (int t0 = 4 * me; t0 < p.max_tokens; t0 += 4 * everyone) {
        long long slot[4] = {-1, -1, -1, -1}, position[4] = {0, 0, 0, 0};
        int row[4] = {-1, -1, -1, -1};
        if (t0 < offset[R]) {
            int low = 0, high = R;  // offset[low] <= t0 < offset[high]
            while (high - low > 1) {
                const int middle = (low + high) >> 1;
                if (offset[middle] <= t0)
                    low = middle;
                else
                    high = middle;
            }
            int loaded = -1, entry = -1;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (t0 + i >= offset[R]) break;
                while (offset[low + 1] <= t0 + i) {
                    ++low;
                    loaded = -1;
                }
                const int at = kept_tokens[low] + t0 + i - offset[low];
                if (at >> p.page_shift != loaded) {
                    loaded = at >> p.page_shift;
                    entry = __ldcg(p.table + static_cast<size_t>(low) * p.width + loaded);
                }
                if (entry >= 0 && entry < p.pages)
                    slot[i] = (static_cast<long long>(entry) << p.page_shift) + (at & (page - 1));
                position[i] = at;
                row[i] = low;
            }
        }
        if (t0 + 4 <= p.max_tokens) {
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                *reinterpret_cast<longlong2*>(p.slots + t0 + i) = make_longlong2(slot[i], slot[i + 1]);
                *reinterpret_cast<longlong2*>(p.positions + t0 + i) = make_longlong2(position[i], position[i + 1]);
            }
            *reinterpret_cast<int4*>(p.rows + t0) = make_int4(row[0], row[1], row[2], row[3]);
        } else {
            for (int i = 0; t0 + i < p.max_tokens; ++i) {
                p.slots[t0 + i] = slot[i];
                p.positions[t0 + i] = position[i];
                p.rows[t0 + i] = row[i];
            }
        }
    }
}

// ---------------------------------------------------------------------------------------
// Keys and values into their slots: 16 bytes a thread.  HBM bounds it: 16,384 tokens of 8 heads of 128, an eighth of them
// without a slot, take 20.0 us, 5.9 TB/s (floor 18.0); one token 1.4 us.
// ---------------------------------------------------------------------------------------
struct AppendArgs {
    int tokens, kv_heads, vectors;   // vectors: of 16 bytes in a head's row
    int page_shift;
    long long slots_end;
    Strides2 key, value;
    Strides3 kpool, vpool;
    const unsigned short *k, *v;
    unsigned short *key_pages, *value_pages;
    const long long* slots;
};

__global__ void __launch_bounds__(256) append_kernel(const AppendArgs p) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const long long per_token = static_cast<long long>(p.kv_heads) * p.vectors;
    const long long all = per_token * p.tokens;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < all; i += gridDim.x * 256ll) {
        const int t = static_cast<int>(i / per_token), rest = static_cast<int>(i % per_token);
        const int h = rest / p.vectors, c = rest % p.vectors * 8;
        const long long slot = p.slots[t];
        if (slot < 0 || slot >= p.slots_end) continue;
        const long long at = slot >> p.page_shift, in_page = slot & ((1 << p.page_shift) - 1);
        const uint4 k = *reinterpret_cast<const uint4*>(p.k + t * p.key.token + h * p.key.head + c);
        const uint4 v = *reinterpret_cast<const uint4*>(p.v + t * p.value.token + h * p.value.head + c);
        *reinterpret_cast<uint4*>(p.key_pages + at * p.kpool.page + in_page * p.kpool.token + h * p.kpool.head + c) = k;
        *reinterpret_cast<uint4*>(p.value_pages + at * p.vpool.page + in_page * p.vpool.token + h * p.vpool.head + c) =
            v;
    }
}

// ---------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------
bool page_size_covered(int page_size) {
    return page_size >= 8 && page_size <= 1024 && (page_size & (page_size - 1)) == 0;
}

int shift_of(int page_size) {
    int shift = 0;
    while ((1 << shift) < page_size) ++shift;
    return shift;
}

// Rows of 16-bit values that the kernels read 16 bytes at a time.
bool aligned(uint64_t address, std::initializer_list<int64_t> strides) {
    if (address % 16 != 0) return false;
    for (const int64_t s : strides)
        if (s < 0 || s % 8 != 0) return false;
    return true;
}

int attention_args(const mb_paged_attention_args* a, bool prefill, AttentionArgs& p) {
    if (a == nullptr) return MB_ERR_INVALID;
    if (a->tokens < 1 || a->requests < 1 || a->kv_heads < 1 || a->heads < 1 || a->heads % a->kv_heads != 0 ||
        a->width < 1 || a->pages < 1 || a->query == 0 || a->key_pages == 0 || a->value_pages == 0 || a->block_table == 0 ||
        a->lengths == 0 || a->out == 0 || (a->key == 0) != (a->value == 0) ||
        (prefill && (a->index == 0 || a->key != 0)) || a->wait_limit_ns < 0)
        return MB_ERR_INVALID;
    if ((a->element != MB_BF16 && a->element != MB_FP16) || !page_size_covered(a->page_size) ||
        (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256) ||
        static_cast<int64_t>(a->width) * a->page_size > kMaxTokens)
        return MB_ERR_UNSUPPORTED;
    if (!aligned(a->query, {a->query_token, a->query_head}) || !aligned(a->out, {}) ||
        !aligned(a->key_pages, {a->kpool_page, a->kpool_token, a->kpool_head}) ||
        !aligned(a->value_pages, {a->vpool_page, a->vpool_token, a->vpool_head}) ||
        (a->key != 0 && (!aligned(a->key, {a->key_token, a->key_head}) ||
                         !aligned(a->value, {a->value_token, a->value_head}))) ||
        a->block_table % 4 || a->lengths % 4 || a->index % 4 || a->status % 4)
        return MB_ERR_INVALID;
    if (a->requests > kMaxRows) return MB_ERR_UNSUPPORTED;
    p.tokens = a->tokens;
    p.requests = a->requests;
    p.heads = a->heads;
    p.kv_heads = a->kv_heads;
    p.head_dim = a->head_dim;
    p.width = a->width;
    p.pages = a->pages;
    p.page_shift = shift_of(a->page_size);
    p.zero_rest = a->zero_rest;
    p.scale = a->scale;
    p.q = {a->query_token, a->query_head};
    p.k = {a->key_token, a->key_head};
    p.v = {a->value_token, a->value_head};
    p.kpool = {a->kpool_page, a->kpool_token, a->kpool_head};
    p.vpool = {a->vpool_page, a->vpool_token, a->vpool_head};
    p.query = reinterpret_cast<const unsigned short*>(a->query);
    p.key = reinterpret_cast<const unsigned short*>(a->key);
    p.value = reinterpret_cast<const unsigned short*>(a->value);
    p.key_pages = reinterpret_cast<const unsigned short*>(a->key_pages);
    p.value_pages = reinterpret_cast<const unsigned short*>(a->value_pages);
    p.table = reinterpret_cast<const int*>(a->block_table);
    p.lengths = reinterpret_cast<const int*>(a->lengths);
    p.index = reinterpret_cast<const int*>(a->index);
    p.out = reinterpret_cast<unsigned short*>(a->out);
    p.status = reinterpret_cast<int*>(a->status);
    p.wait_limit_ns = a->wait_limit_ns != 0 ? a->wait_limit_ns : static_cast<int>(kPipeTimeoutNs);
    return prefill ? prompt_admitted(p) : decode_admitted(p);
}

}  // namespace paged
}  // namespace mb

extern "C" {

int mb_paged_reserve(const mb_paged_reserve_args* a, void* stream) {
    using namespace mb::paged;
    if (a == nullptr || a->requests < 1 || a->width < 1 || a->pages < 1 || a->max_tokens < 0 || a->counts == 0 ||
        a->lengths == 0 || a->block_table == 0 || a->free_pages == 0 || a->free_count == 0 || a->offsets == 0 ||
        a->granted == 0 || (a->max_tokens > 0 && (a->slots == 0 || a->positions == 0 || a->rows == 0)))
        return MB_ERR_INVALID;
    if ((a->counts | a->lengths | a->block_table | a->free_pages | a->free_count | a->offsets | a->granted) % 4 ||
        (a->slots | a->positions | a->rows) % 16)
        return MB_ERR_INVALID;
    if (a->requests > kMaxRows || a->max_tokens > kMaxTokens || !page_size_covered(a->page_size) ||
        static_cast<int64_t>(a->width) * a->page_size > kMaxTokens ||
        static_cast<int64_t>(a->requests) * a->width > INT32_MAX)   // pages of all rows, whatever the lengths say
        return MB_ERR_UNSUPPORTED;
    ReserveArgs p;
    p.requests = a->requests;
    p.width = a->width;
    p.pages = a->pages;
    p.page_shift = shift_of(a->page_size);
    p.max_tokens = a->max_tokens;
    p.counts = reinterpret_cast<const int*>(a->counts);
    p.lengths = reinterpret_cast<int*>(a->lengths);
    p.table = reinterpret_cast<int*>(a->block_table);
    p.stack = reinterpret_cast<int*>(a->free_pages);
    p.free_count = reinterpret_cast<int*>(a->free_count);
    p.offsets = reinterpret_cast<int*>(a->offsets);
    p.rows = reinterpret_cast<int*>(a->rows);
    p.granted = reinterpret_cast<int*>(a->granted);
    p.slots = reinterpret_cast<long long*>(a->slots);
    p.positions = reinterpret_cast<long long*>(a->positions);
    static_assert((4 * kMaxRows + 1) * 4 <= 47 * 1024, "the rows fit without asking for more shared memory");
    const int smem = (4 * a->requests + 1) * 4;
    const cudaError_t err =
        a->max_tokens > 1024 || a->requests > 64
            ? launch_early(reserve_kernel<512>, dim3(kReserveCluster), 512, smem, kReserveCluster,
                           static_cast<cudaStream_t>(stream), p)
            : launch_early(reserve_kernel<128>, dim3(1), 128, smem, 1, static_cast<cudaStream_t>(stream), p);
    return err == cudaSuccess ? MB_OK : mb::cuda_error(err, "mb_paged_reserve");
}

int mb_paged_append(const mb_paged_append_args* a, void* stream) {
    using namespace mb::paged;
    if (a == nullptr || a->tokens < 1 || a->kv_heads < 1 || a->pages < 1 || a->key == 0 || a->value == 0 ||
        a->key_pages == 0 || a->value_pages == 0 || a->slots == 0 || a->slots % 8)
        return MB_ERR_INVALID;
    if (!page_size_covered(a->page_size) || (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256))
        return MB_ERR_UNSUPPORTED;
    if (!aligned(a->key, {a->key_token, a->key_head}) || !aligned(a->value, {a->value_token, a->value_head}) ||
        !aligned(a->key_pages, {a->kpool_page, a->kpool_token, a->kpool_head}) ||
        !aligned(a->value_pages, {a->vpool_page, a->vpool_token, a->vpool_head}))
        return MB_ERR_INVALID;
    AppendArgs p;
    p.tokens = a->tokens;
    p.kv_heads = a->kv_heads;
    p.vectors = a->head_dim / 8;
    p.page_shift = shift_of(a->page_size);
    p.slots_end = static_cast<long long>(a->pages) * a->page_size;
    p.key = {a->key_token, a->key_head};
    p.value = {a->value_token, a->value_head};
    p.kpool = {a->kpool_page, a->kpool_token, a->kpool_head};
    p.vpool = {a->vpool_page, a->vpool_token, a->vpool_head};
    p.k = reinterpret_cast<const unsigned short*>(a->key);
    p.v = reinterpret_cast<const unsigned short*>(a->value);
    p.key_pages = reinterpret_cast<unsigned short*>(a->key_pages);
    p.value_pages = reinterpret_cast<unsigned short*>(a->value_pages);
    p.slots = reinterpret_cast<const long long*>(a->slots);
    const long long blocks = (static_cast<long long>(a->tokens) * a->kv_heads * p.vectors + 255) / 256;
    const cudaError_t err = launch_early(append_kernel, dim3(static_cast<int>(blocks < 148 * 8 ? blocks : 148 * 8)), 256, 0, 1,
                                         static_cast<cudaStream_t>(stream), p);
    return err == cudaSuccess ? MB_OK : mb::cuda_error(err, "mb_paged_append");
}

int64_t mb_paged_attention_workspace(const mb_paged_attention_args* a) {
    mb::paged::AttentionArgs p;
    const int rc = mb::paged::attention_args(a, false, p);
    return rc == MB_OK ? mb::paged::decode_workspace(p) : -rc;
}

int mb_paged_attention(const mb_paged_attention_args* a, void* stream) {
    mb::paged::AttentionArgs p;
    const int rc = mb::paged::attention_args(a, false, p);
    if (rc != MB_OK) return rc;
    return mb::paged::decode_attention(p, a->element, reinterpret_cast<void*>(a->workspace),
                                       static_cast<cudaStream_t>(stream));
}

int64_t mb_paged_prefill_workspace(const mb_paged_attention_args* a) {
    mb::paged::AttentionArgs p;
    const int rc = mb::paged::attention_args(a, true, p);
    return rc == MB_OK ? mb::paged::prompt_workspace(p) : -rc;
}

int mb_paged_prefill(const mb_paged_attention_args* a, void* stream) {
    mb::paged::AttentionArgs p;
    const int rc = mb::paged::attention_args(a, true, p);
    if (rc != MB_OK) return rc;
    return mb::paged::prompt_attention(p, a->element, reinterpret_cast<void*>(a->workspace),
                                       static_cast<cudaStream_t>(stream));
}

}  // extern "C"
