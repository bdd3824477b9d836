// Causal attention of several new tokens a request over a paged key-value cache (mb_paged_prefill): the formula of
// mb_paged_decode.cu for every query, whose position is the last key that it sees.
//
// Tensor cores bound it: 4 head_dim operations a pair of a query and a key it sees.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cstdint>

#include "mb_device.cuh"
#include "mb_kernels.h"
#include "mb_paged.cuh"
#include "mb_tensor.cuh"

namespace mb {
namespace paged {
namespace {

constexpr int kRows = 128;             // of a query tile: tokens times the query heads of a key head
constexpr int kThreads = 384;          // 4 + 4 softmax warps, one that copies, two that issue products, one that cleans
constexpr int kBlock = 64;             // keys of a block
constexpr int kMaxTiles = 12;          // of the ring: keys and values in turn
constexpr int kInfos = 16;             // blocks whose masks are kept
constexpr int kSmemLimit = 227 * 1024;
// What a unit costs besides its keys, in keys: its outputs, and the way from one to the next.  With 128 and 256, 8,192
// tokens of 128-wide heads took 510 and 481 us (192: 492, 320: 484), seven prompts of 64-wide ones 72 and 78.
__host__ __device__ constexpr int tile_cost(int head_dim) { return head_dim == 64 ? 128 : 256; }
// Keys of a run at least, where units are cut.  A prompt of 1,000 tokens, 9/3 heads of 64: 128 keys 21.3 us, 256 21.8, 512
// 24.2; 300 tokens after 2,000: 21.5, 20.5, 24.2; 64 after 3,000, 32/8 heads of 128: 29.5, 28.6, 30.0 (before the join
// took less).
constexpr int kLeastKeys = 256;
// Rows of the table that hold no more are not cut, whatever lengths are, which the host does not know: one launch and no
// scratch (19 tokens: 9.2 to 9.7 us in a table of 4 pages of 64, 14.4 to 15.2 in one of 128).  Rows of up to 1,024 keys:
// 8 x 40 tokens after 700 uncut 27.9 us, cut 24.7; 4 x 600 36.2 and 34.0; one of 500 18.8 and 20.5.
constexpr int kWholeKeys = 512;
constexpr unsigned int kTmemColumns = 512;
// A row's maximum may lag behind by this many powers of two before its sums are rescaled.
constexpr float kLag = 8.f;
// Keys of a block whose exponentials are done when the turn passes to the other tile's warp (8,192 tokens of 128-wide heads:
// 520 us at the end of the block, 505 anywhere from 40 on; 517 without turns where it is 490 with them: both warps of a
// scheduler then do their exponentials at the same time, and everything else).
constexpr int kPassAt = 48;
// As kWeightShift, with room for the lag.
template <typename T>
constexpr float kPromptShift = 7.f;
template <>
constexpr float kPromptShift<__nv_bfloat16> = -39.f;

template <int D>
struct Config {
    static constexpr int kTiles = D == 256 ? 1 : 2;          // query tiles that share a block
    static constexpr int kChunks = D / 64;                   // 128-byte columns
    static constexpr int kQueryBytes = kRows * D * 2;        // of one query tile
    static constexpr int kTileBytes = kBlock * D * 2;        // of a block's keys, and of its values
    static constexpr int kColumnO = 2 * kTiles * kBlock;     // tensor memory: two slots of scores a tile, then the outputs
};

// What a CTA leaves behind about the unit that it began and others finish.
struct Split {
    int first, head, tokens, pieces;
};

struct PromptArgs {
    AttentionArgs a;
    int tile_tokens;       // of one query tile
    int ring;              // tiles
    float scale_log2;
    Split* splits;         // [ctas]
    float* stats;          // [ctas][2][tiles * 128][2]
    float* partial;        // [ctas][2][D / 4][tiles * 128][4]
};

// A piece of a unit, as the warp that copies tells the others.
struct Work {
    int request, head;
    int begin, end, blocks;      // blocks of this piece, and of the unit; end < 0: nothing more
    int first, tokens;           // queries of the unit
    int position;                // of its first query
    int stop0;                   // end of the blocks that its first query tile takes part in
    int alone;                   // one query tile of two
    int pieces;                  // CTAs that the unit's keys are shared out to, from this one on
    int counted;                 // an empty piece that is one of another CTA's `pieces`
};
constexpr int kQueue = 4;
// What is special about a block: keys of it do not count, or some queries of the unit come before keys of it.
constexpr int kMasked = 1, kDiagonal = 2;
constexpr int kStaging = 32 * 64;    // of a softmax warp's outputs

struct Waits {
    int abort_flag;              // one of the CTA's ran out
    int limit_ns;
};

struct PromptControl {
    Work work[kQueue];
    unsigned long long work_full[kQueue], work_empty[kQueue];
    unsigned long long full[kMaxTiles], empty[kMaxTiles], clean[kMaxTiles];
    unsigned long long q_full, q_empty, s_full[4], p_full[4], pv_done[4], o_empty[2];   // [slot], [tile] the last
    unsigned long long half_ready, half_taken;
    unsigned long long turn[2][4];   // [query tile][warp]: its exponentials
    float half[kRows][2];        // maximum and sum of the second half of a lone query tile's keys
    unsigned int mask[kInfos][2];
    int special[kInfos];         // of a block: kMasked, kDiagonal
    int odd[kInfos];             // values that are no numbers were taken out of it
    long long warp_sums[kThreads / 32];
    unsigned int tmem;
    Waits waits;
};

struct Request {
    int first, tokens, length;   // its queries, and its keys
};

// ---------------------------------------------------------------------------------------
// The deal: units (a request, a key head, a pair of query tiles) one after the other, each as long as the keys its last
// query sees and a constant, in equal runs over the CTAs.  A run begins and ends anywhere in a unit, at the nearest
// block.  Lengths before a unit of a request are an arithmetic series, so a place is found by bisection.
// ---------------------------------------------------------------------------------------
struct Deal {
    const long long* before;     // [requests + 1] lengths of the requests before, for one head
    const Request* requests;
    int count, heads, unit_tokens, cost;
    long long total, per;
};

__device__ __forceinline__ int units_of(const Request& q, int unit_tokens) {
    return (q.tokens + unit_tokens - 1) / unit_tokens;
}
// Lengths of the first `j` of the request's units, all of them full.
__device__ __forceinline__ long long length_before(const Request& q, int unit_tokens, int cost, long long j) {
    return j * (max(q.length - q.tokens, 0) + cost) + j * (j + 1) / 2 * unit_tokens;
}
__device__ __forceinline__ long long request_length(const Request& q, int unit_tokens, int cost) {
    const int units = units_of(q, unit_tokens);
    if (units == 0) return 0;
    return length_before(q, unit_tokens, cost, units - 1) + max(q.length - q.tokens, 0) + q.tokens + cost;
}

struct Piece {
    int request, head;
    int begin, end, blocks;      // blocks of this piece, and of the unit
    int first, tokens;           // queries of the unit
    int position;                // of its first query
    long long unit_end;          // in the deal
    long long next;              // where this piece ends in the deal
    bool at_start;               // of the unit

    // Not inlined: the arithmetic of one piece is as much code as a softmax warp's loop, which it would drive out of the
    // instruction cache.
    __device__ __noinline__ Piece(const Deal& d, long long at, long long run_end) {
        int low = 0, high = d.count;   // before[low] * heads <= at < before[high] * heads
        while (high - low > 1) {
            const int middle = (low + high) >> 1;
            if (d.before[middle] * d.heads <= at)
                low = middle;
            else
                high = middle;
        }
        request = low;
        const Request q = d.requests[low];
        const long long length = d.before[low + 1] - d.before[low];
        long long rest = at - d.before[low] * d.heads;
        head = static_cast<int>(rest / length);
        rest -= head * length;
        int units = units_of(q, d.unit_tokens);
        int lower = 0, upper = units;
        while (upper - lower > 1) {
            const int middle = (lower + upper) >> 1;
            if (length_before(q, d.unit_tokens, d.cost, middle) <= rest)
                lower = middle;
            else
                upper = middle;
        }
        const int tile = lower;
        const long long start = length_before(q, d.unit_tokens, d.cost, tile);
        const long long end_of = tile + 1 == units ? length : length_before(q, d.unit_tokens, d.cost, tile + 1);
        const long long unit_begin = at - (rest - start);
        unit_end = unit_begin + (end_of - start);
        next = min(unit_end, run_end);
        first = q.first + tile * d.unit_tokens;
        tokens = min(q.tokens - tile * d.unit_tokens, d.unit_tokens);
        position = q.length - q.tokens + tile * d.unit_tokens;
        blocks = max((position + tokens + kBlock - 1) / kBlock, 1);
        begin = block_at(at - unit_begin, end_of - start);
        end = block_at(next - unit_begin, end_of - start);
        at_start = rest == start;
    }
    __device__ __forceinline__ int block_at(long long offset, long long length) const {
        if (offset >= length) return blocks;
        return static_cast<int>(min((offset + kBlock / 2) / kBlock, static_cast<long long>(blocks)));
    }
};

// The first end or begin of a unit from `at` on.
__device__ __forceinline__ long long unit_boundary(const Deal& d, long long at) {
    if (at >= d.total) return at;
    const Piece u(d, at, d.total);
    return u.at_start ? at : u.unit_end;
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z,
                                            unsigned long long* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void tma_load_column(void* dst, const CUtensorMap* map, int column, int place, int head, int page,
                                                unsigned long long* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(dst)),
        "l"(map), "r"(column), "r"(place), "r"(head), "r"(page), "r"(smem_u32(bar))
        : "memory");
}
// D[tmem] (+)= A[tmem] . B[smem]: A's 16-bit elements two to a column, a row a lane.
__device__ __forceinline__ void umma_from_tmem(unsigned int tmem_d, unsigned int tmem_a, unsigned long long desc_b,
                                               unsigned int idesc, unsigned int accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
        "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Shared-memory operand whose rows are the reduction: [column of 64 elements][row], 128-byte swizzle; rows in groups of
// 8 that lie 1024 bytes apart, columns `column_bytes` apart.
__device__ __forceinline__ unsigned long long umma_desc_rows(unsigned int smem_addr, unsigned int column_bytes) {
    unsigned long long d = 0;
    d |= static_cast<unsigned long long>((smem_addr & 0x3ffffu) >> 4);
    d |= static_cast<unsigned long long>(column_bytes >> 4) << 16;
    d |= static_cast<unsigned long long>(1024 >> 4) << 32;
    d |= 1ull << 46;
    d |= 2ull << 61;
    return d;
}
// 32 columns of this thread's lane, not waited for.
__device__ __forceinline__ void tmem_load32_async(unsigned int taddr, float* v) {
    unsigned int* r = reinterpret_cast<unsigned int*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
          "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
          "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_store16(unsigned int taddr, const unsigned int (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// Two floats in a 64-bit register, for instructions that work on both.
__device__ __forceinline__ unsigned long long pair_of(float x, float y) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float pair_low(unsigned long long v) { return __uint_as_float(static_cast<unsigned int>(v)); }
__device__ __forceinline__ float pair_high(unsigned long long v) {
    return __uint_as_float(static_cast<unsigned int>(v >> 32));
}
__device__ __forceinline__ unsigned long long fma_pair(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ unsigned long long add_pair(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

template <typename T>
__device__ __forceinline__ unsigned int pack_pair(float x, float y) {
    if constexpr (std::is_same_v<T, __half>) {
        const __half2 h = __floats2half2_rn(x, y);
        return *reinterpret_cast<const unsigned int*>(&h);
    } else {
        return prefill::pack_bf16_pair(x, y);
    }
}

// Whether one of two 16-bit values is infinite or NaN: all bits of its exponent set, which one more carries out of it.
template <typename T>
__device__ __forceinline__ bool not_finite(unsigned int v) {
    constexpr unsigned int kExponents = std::is_same_v<T, __half> ? 0x7c007c00u : 0x7f807f80u;
    constexpr unsigned int kOnes = std::is_same_v<T, __half> ? 0x04000400u : 0x00800080u;
    return ((v & kExponents) + kOnes & 0x80008000u) != 0u;
}
template <typename T>
__device__ __forceinline__ unsigned int without_odd(unsigned int v) {
    return (not_finite<T>(v & 0xffffu) ? 0u : v & 0xffffu) | (not_finite<T>(v & 0xffff0000u) ? 0u : v & 0xffff0000u);
}
// The infinities and NaN that were taken out of blocks `from` .. `stop` - 1 of a unit, 32 columns of them from `column` on,
// added to the outputs of a query at `position`.  `info` is that of block `end`.
template <typename T>
__device__ __noinline__ void give_back(float* o, const AttentionArgs& a, const PromptControl* ctl, const Work* u, int info,
                                       int from, int stop, int end, int column, int position) {
#pragma unroll 1
    for (int b = from; b < stop; ++b) {
        const int block_info = (info + 2 * kInfos - (end - b)) % kInfos;
        if (ctl->odd[block_info] == 0) continue;
#pragma unroll 1
        for (int k = 0; k < kBlock; ++k) {
            const int key = b * kBlock + k;
            if (!((ctl->mask[block_info][k >> 5] >> (k & 31)) & 1u) || key > position) continue;
            const long long entry = a.table[static_cast<size_t>(u->request) * a.width + (key >> a.page_shift)];
            const unsigned short* values = a.value_pages + entry * a.vpool.page +
                                           (key & ((1 << a.page_shift) - 1)) * a.vpool.token + u->head * a.vpool.head + column;
#pragma unroll 1
            for (int i = 0; i < 32; ++i) {
                const unsigned short bits = values[i];
                if (!not_finite<T>(bits)) continue;
                if constexpr (std::is_same_v<T, __half>)
                    o[i] += __half2float(*reinterpret_cast<const __half*>(&bits));
                else
                    o[i] += bf16_bits_to_float(bits);
            }
        }
    }
}

// Bounded waits.  What a wait that does not succeed at once does is one function for all of them: inlined into every one
// it is a good part of the code that has to stay in the instruction cache.
__device__ __noinline__ bool wait_on(unsigned long long* bar, unsigned int parity, volatile Waits* waits) {
    return wait_within(bar, parity, &waits->abort_flag, waits->limit_ns);
}
__device__ __forceinline__ bool wait_thread(unsigned long long* bar, unsigned int parity, volatile Waits* waits) {
    return mbar_try_wait(bar, parity) || wait_on(bar, parity, waits);
}
// Of a whole warp.
__device__ __forceinline__ bool wait_warp(unsigned long long* bar, unsigned int parity, volatile Waits* waits) {
    return __all_sync(0xffffffffu, wait_thread(bar, parity, waits)) != 0;
}

// ---------------------------------------------------------------------------------------
// The kernel.  Two query tiles of 128 rows (tokens x the query heads of a key head) share every block of 64 keys, and
// every tile has two slots of scores in tensor memory: while its softmax warps work on one block, the scores of the
// next are there or under way, and the tensor core multiplies for both tiles.  Weights go back to tensor memory as
// 16-bit numbers over the scores they were made of and are the first operand of the second product, values are taken
// as they lie in the pages (rows are the reduction).  A thread has a row: no shuffles.  Outputs stay in tensor
// memory and are rescaled only when a row's maximum has grown by more than 2^8 since the last time.  256-wide
// heads: one query tile.
//
// A weight is one 16-bit number in the second product, off by up to half a step of its type, while the sum below it has 32 bits.
// Errors against 64 bits (2-norm) are 0.0017 to 0.0023 for bf16, of which rounding the output is 0.0015 to 0.0017; a second
// number, as decode has, would be half as many products again in the kernel that they bound.  fp16 weights are 2^7 to 2^15
// at the maximum: one of 2^-21 of it and less has fewer digits, one below 2^-32 none.
//
// Measured (us; floor at the measured GEMM rate): 8,192 tokens, 32/8 heads of 128: 570 to 581 a pass among many (332), 0.95
// PFLOP/s, at the power limit; 497 to 521 in a graph of few, 1.08 PFLOP/s; 509 tokens after 16,000, 8/1 heads of 256: 84 to 88
// (41); seven prompts of up to 1,031, 32/8 heads of 64, pages of 16: 59 (8).
//
// What bounds it: a block of 64 keys takes 1,700 to 1,900 cycles, of which the exponentials of its two tiles, 8 cycles a warp and instruction, are 1,024, and the products 1,280 (64 keys a product of scores read the queries from shared
// memory for 64 columns, at two thirds of the rate that 128 columns reach); between units there are the
// outputs.  Blocks of 128 keys leave one slot a tile, and the chain scores -> weights -> outputs -> scores of a tile then
// takes 3,300 cycles (558 us).  A quarter to five eighths of the exponentials by a polynomial on the multipliers took 562
// to 675 us instead of 553.  The code matters as much: a third less of it around the same loops was worth 520 -> 508 us.
// ---------------------------------------------------------------------------------------
template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
prompt_attention_kernel(const __grid_constant__ CUtensorMap query_map, const __grid_constant__ CUtensorMap key_map,
                        const __grid_constant__ CUtensorMap value_map, const __grid_constant__ PromptArgs p) {
    using C = Config<D>;
    constexpr int kTiles = C::kTiles, kChunks = C::kChunks;
    extern __shared__ __align__(1024) unsigned char smem[];
    unsigned char* queries = smem;                                   // [tiles][chunks][128 rows][128 bytes]
    unsigned char* ring = queries + kTiles * C::kQueryBytes;         // [ring][chunks][block rows][128 bytes]
    unsigned char* stagings = ring + static_cast<size_t>(p.ring) * C::kTileBytes;   // [softmax warps][32 rows][64 bytes]
    PromptControl* ctl = reinterpret_cast<PromptControl*>(stagings + kTiles * 4 * kStaging);
    long long* before = reinterpret_cast<long long*>(ctl + 1);       // [requests + 1]
    Request* requests = reinterpret_cast<Request*>(before + p.a.requests + 1);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int shift = p.a.page_shift, page = 1 << shift;
    const int group = p.a.heads / p.a.kv_heads;
    if (tid == 0) {
        for (int s = 0; s < p.ring; ++s) {
            mbar_init(&ctl->full[s], 1);
            mbar_init(&ctl->empty[s], kTiles + 1);
            mbar_init(&ctl->clean[s], 1);
        }
        mbar_init(&ctl->q_full, 1);
        mbar_init(&ctl->q_empty, kTiles);
        for (int s = 0; s < 4; ++s) {
            mbar_init(&ctl->s_full[s], 1);
            mbar_init(&ctl->p_full[s], 4);
            mbar_init(&ctl->pv_done[s], 1);
        }
        mbar_init(&ctl->o_empty[0], 4);
        mbar_init(&ctl->o_empty[1], 4);
        for (int q = 0; q < kQueue; ++q) {
            mbar_init(&ctl->work_full[q], 1);
            mbar_init(&ctl->work_empty[q], 5 * kTiles + 1);   // warps of softmax, of products, and the one that cleans
        }
        for (int w = 0; w < 8; ++w) mbar_init(&ctl->turn[w >> 2][w & 3], 1);
        mbar_init(&ctl->half_ready, 4);
        mbar_init(&ctl->half_taken, 4);
        ctl->waits.abort_flag = 0;
        ctl->waits.limit_ns = p.a.wait_limit_ns;
        mbar_init_fence();
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // Not before the wait: the kernel that it is for may be anybody's, and one that let this launch begin before it allocated
    // would wait for these columns.  For the same reason the next launch may begin only when they are taken.
    if (warp == 11) prefill::tmem_alloc(&ctl->tmem, kTmemColumns);
    prefill::tc_fence_before();
    __syncthreads();
    prefill::tc_fence_after();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const unsigned int tmem = ctl->tmem;

    Deal deal;
    deal.before = before;
    deal.requests = requests;
    deal.count = p.a.requests;
    deal.heads = p.a.kv_heads;
    deal.unit_tokens = p.tile_tokens * kTiles;
    deal.cost = tile_cost(D);
    {
        const int each = (p.a.requests + kThreads - 1) / kThreads;
        const int r0 = min(tid * each, p.a.requests), r1 = min(r0 + each, p.a.requests);
        const int capacity = p.a.width << shift;
        long long sum = 0;
        for (int r = r0; r < r1; ++r) {
            const int first = min(max(p.a.index[r], 0), p.a.tokens), end = min(max(p.a.index[r + 1], first), p.a.tokens);
            const Request q = {first, end - first, min(max(p.a.lengths[r], 0), capacity)};
            requests[r] = q;
            sum += request_length(q, deal.unit_tokens, deal.cost);
        }
        long long inclusive = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const long long other = __shfl_up_sync(0xffffffffu, inclusive, d);
            if (lane >= d) inclusive += other;
        }
        if (lane == 31) ctl->warp_sums[warp] = inclusive;
        __syncthreads();
        long long mine = inclusive - sum;
        for (int w = 0; w < warp; ++w) mine += ctl->warp_sums[w];
        for (int r = r0; r < r1; ++r) {
            before[r] = mine;
            mine += request_length(requests[r], deal.unit_tokens, deal.cost);
        }
        if (r0 < p.a.requests && r1 == p.a.requests) before[p.a.requests] = mine;
        __syncthreads();
    }
    deal.total = before[p.a.requests] * deal.heads;
    deal.per = max((deal.total + gridDim.x - 1) / gridDim.x, p.splits != nullptr ? static_cast<long long>(kLeastKeys) : 1);
    long long run_begin = min(blockIdx.x * deal.per, deal.total);
    long long run_end = min(run_begin + deal.per, deal.total);
    if (p.splits == nullptr) {   // no unit is cut: runs go from unit to unit
        run_begin = unit_boundary(deal, run_begin);
        run_end = unit_boundary(deal, run_end);
    }
    volatile Waits* waits = &ctl->waits;
    bool ok = true;

    // The next piece, for a warp that all comes to; it keeps what it needs of it, or lets go of it later.
    int queue = 0;
    unsigned int queue_round = 0;
    auto next_work = [&]() -> const Work* {
        ok = ok && wait_warp(&ctl->work_full[queue], queue_round & 1, waits);
        return ok && ctl->work[queue].end >= 0 ? &ctl->work[queue] : nullptr;
    };
    auto release_work = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl->work_empty[queue]);
        if (++queue == kQueue) {
            queue = 0;
            ++queue_round;
        }
    };

    if (warp == 8) {
        // ---- copies
        int stage = 0, info = 0;
        unsigned int round = 0, units = 0;
        constexpr int kBlockShift = 6;
        static_assert(1 << kBlockShift == kBlock);
        const int rows_shift = min(shift, kBlockShift), rows = 1 << rows_shift;
        const int per_shift = kBlockShift - rows_shift, per_block = 1 << per_shift;   // table entries of a block
        const int batch = 32 >> per_shift;                                            // blocks whose entries the lanes hold
        long long at = run_begin;
        // a piece ahead of the copies, so that nobody waits for the arithmetic
        auto publish = [&]() {
            if (queue_round > 0)
                ok = wait_warp(&ctl->work_empty[queue], (queue_round - 1) & 1, waits);
            if (!ok) return;
            Work w = {};
            w.end = -1;
            if (at < run_end) {
                // A unit of two query tiles: each takes the blocks up to the one its last query lies in.  A lone tile of a pair
                // takes the place of both, which share its blocks in turn and meet at the end.
                const Piece u(deal, at, run_end);
                at = u.next;
                w.request = u.request;
                w.head = u.head;
                w.begin = u.begin;
                w.end = u.end;
                w.blocks = u.blocks;
                w.first = u.first;
                w.tokens = u.tokens;
                w.position = u.position;
                w.alone = kTiles == 2 && u.tokens <= p.tile_tokens;
                w.stop0 = kTiles == 1 || w.alone
                              ? u.end
                              : min(max((u.position + p.tile_tokens + kBlock - 1) / kBlock, 1), u.end);
                w.pieces = static_cast<int>((u.unit_end - 1) / deal.per - blockIdx.x) + 1;
                w.counted = !u.at_start;
            }
            if (lane == 0) {
                ctl->work[queue] = w;
                mbar_arrive(&ctl->work_full[queue]);
            }
            __syncwarp();
            if (++queue == kQueue) {
                queue = 0;
                ++queue_round;
            }
        };
        publish();
        for (int mine_at = 0; ok; mine_at = (mine_at + 1) % kQueue) {
            const Work u = ctl->work[mine_at];
            if (u.end < 0) break;
            publish();
            if (!ok) break;
            if (u.begin >= u.end) continue;
            if (units > 0) ok = wait_warp(&ctl->q_empty, (units - 1) & 1, waits);
            if (!ok) break;
            ++units;
            const int tiles = kTiles == 2 && !u.alone ? 2 : 1;
            if (elect_one()) {
                mbar_arrive_expect_tx(&ctl->q_full, tiles * kChunks * p.tile_tokens * group * 128);
#pragma unroll 1
                for (int t = 0; t < tiles; ++t)
#pragma unroll 1
                    for (int c = 0; c < kChunks; ++c)
                        tma_load_3d(queries + t * C::kQueryBytes + c * kRows * 128, &query_map, c * 64, u.head * group,
                                    u.first + t * p.tile_tokens, &ctl->q_full);
            }
            __syncwarp();
            const int n = max(min(u.position + u.tokens, p.a.width << shift), 0);   // keys that the unit sees
            const int* entries = p.a.table + static_cast<size_t>(u.request) * p.a.width;
            const int entries_end = (n + page - 1) >> shift;
            auto entry_of = [&](int block) {
                const int b = block + (lane >> per_shift);
                const int e = (b * kBlock + ((lane & (per_block - 1)) << rows_shift)) >> shift;
                const int id = b < u.end && e < entries_end ? entries[e] : -1;
                return id >= 0 && id < p.a.pages ? id : -1;
            };
            int next = entry_of(u.begin);
            for (int b = u.begin; ok && b < u.end;) {
                const int mine = next;
                next = entry_of(b + batch);
                for (int j = 0; ok && j < batch && b < u.end; ++j, ++b) {
                    const int place = page > kBlock ? (b * kBlock) & (page - 1) : 0;
                    const unsigned int valid = __ballot_sync(0xffffffffu, mine >= 0) >> (j << per_shift);
                    const int boxes = __popc(valid & ((2u << (per_block - 1)) - 1));
#pragma unroll 1
                    for (int kind = 0; kind < 2; ++kind) {   // keys, then values
                        if (round > 0) ok = wait_warp(&ctl->empty[stage], (round - 1) & 1, waits);
                        if (!ok) break;
                        if (kind == 0 && lane < kBlock / 32) {
                            // which keys of the block count: on a page, and seen by any query of the unit
                            unsigned int word = 0;
#pragma unroll 1
                            for (int i = 0; i < 32; i += 8)
                                if ((valid >> ((lane * 32 + i) >> rows_shift)) & 1u) word |= 0xffu << i;
                            const int left = n - b * kBlock - lane * 32;
                            if (left < 32) word &= left <= 0 ? 0u : (1u << left) - 1;
                            ctl->mask[info][lane] = word;
                        }
                        __syncwarp();
                        if (kind == 0 && lane == 0)
                            ctl->odd[info] = 0, ctl->special[info] = (boxes != per_block || n - b * kBlock < kBlock ? kMasked : 0) |
                                                 (b * kBlock + kBlock - 1 > u.position ? kDiagonal : 0);
                        __syncwarp();
                        if (elect_one())
                            mbar_arrive_expect_tx(&ctl->full[stage], boxes * kChunks * rows * 128);
                        __syncwarp();
                        unsigned char* to = ring + static_cast<size_t>(stage) * C::kTileBytes;
                        const CUtensorMap* map = kind == 0 ? &key_map : &value_map;
                        if (per_block == 1) {
                            const int id = __shfl_sync(0xffffffffu, mine, j);
                            if (id >= 0 && elect_one()) {
#pragma unroll
                                for (int c = 0; c < kChunks; ++c)
                                    tma_load_column(to + c * kBlock * 128, map, c * 64, place, u.head, id, &ctl->full[stage]);
                            }
                        } else {   // a box a lane: a table entry's rows of one 128-byte column
                            const int box = lane & (per_block - 1), column = lane >> per_shift;
                            const int id = __shfl_sync(0xffffffffu, mine, (j << per_shift) + box);
                            if (column < kChunks && id >= 0)
                                tma_load_column(to + (column * kBlock + (box << rows_shift)) * 128, map, column * 64, place,
                                                u.head, id, &ctl->full[stage]);
                        }
                        __syncwarp();
                        if (++stage == p.ring) {
                            stage = 0;
                            ++round;
                        }
                    }
                    info = (info + 1) % kInfos;
                }
            }
        }
    } else if (warp == 9 || (kTiles == 2 && warp == 10)) {
        // ---- products of one query tile.  One thread issues them, in one place for the scores and one for the outputs: what
        // it does between two products is time the tensor core waits, unless the other tile's thread has something for it.
        // (One thread for both tiles was busy 3,000 cycles a block and softmax warps waited 1,900 of them; with a thread a
        // tile a block takes 1,700 to 1,900 and they wait 150.)
        constexpr unsigned int kFormat = std::is_same_v<T, __half> ? 0u : (1u << 7) | (1u << 10);
        constexpr unsigned int kIdescS = (1u << 4) | kFormat | (static_cast<unsigned int>(kBlock >> 3) << 17) |
                                         (static_cast<unsigned int>(kRows >> 4) << 24);
        constexpr unsigned int kIdescO = (1u << 4) | kFormat | (1u << 16) | (static_cast<unsigned int>(D >> 3) << 17) |
                                         (static_cast<unsigned int>(kRows >> 4) << 24);
        if (elect_one()) {
            const int tile = warp - 9;
            const unsigned int ring_at = smem_u32(ring), queries_at = smem_u32(queries);
            // the high half of operand descriptors, and the low ones without the address
            const unsigned int high = static_cast<unsigned int>(prefill::umma_desc(0) >> 32);
            const unsigned int low_rows = static_cast<unsigned int>(umma_desc_rows(0, kBlock * 128));
            const unsigned int low = static_cast<unsigned int>(prefill::umma_desc(0));
            auto descriptor = [&](unsigned int low_half) {
                return static_cast<unsigned long long>(high) << 32 | low_half;
            };
            const unsigned int slots = tmem + tile * 2 * kBlock, outputs = tmem + C::kColumnO + tile * D;
            int key_stage = 0, value_stage = 1, info = 0;    // of the next block
            unsigned int key_round = 0, value_round = 0, units = 0, outputs_used = 0;
            auto advance = [&](int& stage, unsigned int& round) {
                stage += 2;
                if (stage >= p.ring) {
                    stage -= p.ring;
                    ++round;
                }
            };
            unsigned int p_phase = 0;                // bit: slot
            unsigned int clean_phase = 0;            // bit: stage of the ring
            while (ok) {
                ok = wait_thread(&ctl->work_full[queue], queue_round & 1, waits);
                if (!ok) break;
                const int begin = ctl->work[queue].begin, end = ctl->work[queue].end;
                if (end < 0) break;
                const bool alone = ctl->work[queue].alone != 0;
                const int tile_stop = tile == 0 ? ctl->work[queue].stop0 : end;
                mbar_arrive(&ctl->work_empty[queue]);
                if (++queue == kQueue) {
                    queue = 0;
                    ++queue_round;
                }
                if (begin >= end) continue;
                ok = wait_thread(&ctl->q_full, units & 1, waits);
                ++units;
                auto takes = [&](int b) { return alone ? ((b - begin) & 1) == tile : b < tile_stop; };
                const unsigned int q = low + ((queries_at + (alone ? 0 : tile * C::kQueryBytes)) >> 4);
                int bs = begin, bv = begin;          // blocks whose scores, and whose products with values, come next
                unsigned int scored = 0, done = 0;   // steps
                while (ok && bv < end) {
                    if (bs < end && scored - done < 2) {
                        // scores go where the weights of two steps ago were; not waited for while there is something to do
                        const bool idle = bs == bv;
                        if (idle ? ok = wait_thread(&ctl->full[key_stage], key_round & 1, waits)
                                 : mbar_try_wait(&ctl->full[key_stage], key_round & 1)) {
                            if (takes(bs)) {
                                const int slot = scored & 1;
                                const unsigned int k0 = low + ((ring_at + key_stage * C::kTileBytes) >> 4);
                                prefill::tc_fence_after();
#pragma unroll
                                for (int c = 0; c < kChunks; ++c)
#pragma unroll
                                    for (int k = 0; k < 4; ++k)
                                        prefill::umma_bf16(slots + slot * kBlock, descriptor(q + (c * kRows * 128 >> 4) + 2 * k),
                                                           descriptor(k0 + (c * kBlock * 128 >> 4) + 2 * k), kIdescS,
                                                           (c | k) != 0 ? 1u : 0u);
                                prefill::umma_commit(&ctl->s_full[tile * 2 + slot]);
                                prefill::umma_commit(&ctl->empty[key_stage]);
                                ++scored;
                            } else {
                                mbar_arrive(&ctl->empty[key_stage]);
                            }
                            advance(key_stage, key_round);
                            if (++bs == end) prefill::umma_commit(&ctl->q_empty);
                            continue;
                        }
                        if (!ok) break;
                    }
                    ok = wait_thread(&ctl->full[value_stage], value_round & 1, waits);
                    if (ok && takes(bv)) {
                        const int slot = done & 1;
                        if (done == 0 && outputs_used++ > 0)   // the outputs before have been taken
                            ok = wait_thread(&ctl->o_empty[tile], outputs_used & 1, waits);
                        if (ok && ctl->special[info] != 0) {
                            ok = wait_thread(&ctl->clean[value_stage], (clean_phase >> value_stage) & 1, waits);
                            clean_phase ^= 1u << value_stage;
                        }
                        ok = ok && wait_thread(&ctl->p_full[tile * 2 + slot], (p_phase >> slot) & 1, waits);
                        if (!ok) break;
                        p_phase ^= 1u << slot;
                        prefill::tc_fence_after();
                        const unsigned int v = low_rows + ((ring_at + value_stage * C::kTileBytes) >> 4);
#pragma unroll
                        for (int k = 0; k < kBlock / 16; ++k)
                            umma_from_tmem(outputs, slots + slot * kBlock + k * 8, descriptor(v + (k * 16 * 128 >> 4)), kIdescO,
                                           done == 0 && k == 0 ? 0u : 1u);
                        prefill::umma_commit(&ctl->pv_done[tile * 2 + slot]);
                        prefill::umma_commit(&ctl->empty[value_stage]);
                        ++done;
                    } else if (ok) {
                        if (ctl->special[info] != 0) clean_phase ^= 1u << value_stage;
                        mbar_arrive(&ctl->empty[value_stage]);
                    }
                    advance(value_stage, value_round);
                    info = (info + 1) % kInfos;
                    ++bv;
                }
            }
        }
        ok = __all_sync(0xffffffffu, ok);
    } else if (warp == 11) {
        // ---- values of keys that do not count may be anything, and 0 * NaN is NaN: where a block has such keys their rows
        // are zeroed before the product.  Where some queries see a key and some do not, infinities and NaN are taken out and
        // given back to those who see them with the outputs.  Every tile of the ring passes here, so that none is
        // filled again unseen.
        int stage = 0, info = 0;
        unsigned int round = 0;
        while (const Work* u = next_work()) {
            const int blocks = u->end - u->begin;
            release_work();
            for (int b = 0; ok && b < blocks; ++b) {
#pragma unroll 1
                for (int kind = 0; kind < 2; ++kind) {
                    // the one wait that is never suspended, so that a short limit means something: 2 % if all are like that
                    ok = ok && __all_sync(0xffffffffu, mbar_test_wait(&ctl->full[stage], round & 1) ||
                                                           wait_on(&ctl->full[stage], round & 1, waits));
                    if (!ok) break;
                    const int special = kind == 1 ? ctl->special[info] : 0;
                    if (special != 0) {
                        unsigned char* values = ring + static_cast<size_t>(stage) * C::kTileBytes;
                        bool odd = false;
#pragma unroll 2
                        for (int i = lane; i < kBlock * kChunks * 8; i += 32) {
                            const int row = i >> 3 & (kBlock - 1);
                            uint4* at = reinterpret_cast<uint4*>(values + i * 16);
                            if (!((ctl->mask[info][row >> 5] >> (row & 31)) & 1u)) {
                                *at = make_uint4(0u, 0u, 0u, 0u);
                            } else if (special & kDiagonal) {
                                uint4 v = *at;
                                if (not_finite<T>(v.x) | not_finite<T>(v.y) | not_finite<T>(v.z) | not_finite<T>(v.w)) {
                                    odd = true;
                                    v.x = without_odd<T>(v.x);
                                    v.y = without_odd<T>(v.y);
                                    v.z = without_odd<T>(v.z);
                                    v.w = without_odd<T>(v.w);
                                    *at = v;
                                }
                            }
                        }
                        odd = __any_sync(0xffffffffu, odd);
                        if (lane == 0) ctl->odd[info] = odd;
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&ctl->clean[stage]);
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&ctl->empty[stage]);
                    if (++stage == p.ring) {
                        stage = 0;
                        ++round;
                    }
                }
                info = (info + 1) % kInfos;
            }
        }
    } else if (warp < 4 * kTiles) {
        // ---- softmax and outputs of one query tile: a thread has a row
        const int tile = warp >> 2, r = (warp & 3) * 32 + lane;
        const int group_inverse = (65536 + group - 1) / group;   // r / group = r * this >> 16, for r below 128
        const int token = r * group_inverse >> 16;               // of the tile
        const unsigned int lanes = tmem + (static_cast<unsigned int>((warp & 3) * 32) << 16);
        const unsigned int outputs = lanes + C::kColumnO + tile * D;
        int info = 0;
        unsigned int phase = 0;                         // bit: slot
        unsigned int halves = 0;                        // lone tiles so far
        unsigned int turn = 0;                          // turns taken so far
        Split split = {0, 0, 0, 0};
        // The largest score is not that of the largest product.  Otherwise maxima are of products, without the scale.
        const bool premultiply = p.scale_log2 <= 0.f;
        const float multiplier = premultiply ? 1.f : p.scale_log2, lag = kLag / multiplier;
        while (const Work* u = next_work()) {
            const int begin = u->begin, end = u->end;
            if (begin >= end) {
                if (u->counted != 0 && p.splits != nullptr)
                    *reinterpret_cast<float2*>(p.stats + (static_cast<size_t>(blockIdx.x) * 2 * kTiles * kRows +
                                                          tile * kRows + r) * 2) = make_float2(-INFINITY, 0.f);
                release_work();
                continue;
            }
            const bool alone = u->alone != 0;
            const int own = alone ? 0 : tile;                    // query tile
            const int first_block = alone ? begin + tile : begin, blocks = tile == 0 ? u->stop0 : end;
            const int first_position = u->position + own * p.tile_tokens, position = first_position + token;
            // Rows of no query hold whatever lies in shared memory, or the next request's queries: no say in what others do.
            const bool counts = token < min(u->tokens - own * p.tile_tokens, p.tile_tokens);
            float m = -INFINITY, l = 0.f;
            // turns are taken for as many steps as both tiles have
            unsigned int step = 0, turns = 0;
            if constexpr (kTiles == 2) {
                turns = alone ? (end - begin) / 2 : max(u->stop0 - begin, 0);
                if (tile == 1 && turns > 0 && lane == 0) mbar_arrive(&ctl->turn[0][warp & 3]);
            }
            for (int b = first_block; b < blocks; b += alone ? 2 : 1, ++step) {
                const int slot = tile * 2 + (step & 1);
                ok = ok && wait_warp(&ctl->s_full[slot], (phase >> slot) & 1, waits);
                if (!ok) break;
                phase ^= 1u << slot;
                prefill::tc_fence_after();
                const unsigned int scores = lanes + slot * kBlock;
                const int block_info = (info + b - begin) % kInfos;
                const bool partial = (ctl->special[block_info] & kMasked) != 0 || b * kBlock + kBlock - 1 > first_position;
                float s[kBlock];
#pragma unroll
                for (int c = 0; c < kBlock; c += 32) tmem_load32_async(scores + c, s + c);
                tmem_wait_load();
                if (premultiply) {
#pragma unroll
                    for (int c = 0; c < kBlock; ++c) s[c] *= p.scale_log2;
                }
                if (partial) {   // scores that do not count are minus infinity
#pragma unroll
                    for (int w = 0; w < kBlock / 32; ++w) {
                        const int last = position - b * kBlock - w * 32;   // the last key of the word that counts
                        const unsigned int keep =
                            ctl->mask[block_info][w] & (last < 0 ? 0u : last >= 31 ? ~0u : (2u << last) - 1);
#pragma unroll
                        for (int c = 0; c < 32; ++c) s[w * 32 + c] = (keep >> c) & 1u ? s[w * 32 + c] : -INFINITY;
                    }
                }
                float highest[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < kBlock; c += 8)
#pragma unroll
                    for (int i = 0; i < 4; ++i) highest[i] = fmaxf(fmaxf(highest[i], s[c + i]), s[c + 4 + i]);
                const float now = fmaxf(fmaxf(highest[0], highest[1]), fmaxf(highest[2], highest[3]));
                if (b == first_block) {
                    m = now;
                } else if (__any_sync(0xffffffffu, counts && (now > m + lag || (m == -INFINITY && now > m)))) {
                    const float grown = fmaxf(m, now);
                    const float base = grown == -INFINITY ? 0.f : grown;
                    const float factor = prefill::exp2_approx((m - base) * multiplier);
                    m = grown;
                    l *= factor;
                    // the product before is in the outputs; the one before that is, since these scores are there
                    ok = wait_warp(&ctl->pv_done[slot ^ 1], ((phase >> (slot ^ 1)) & 1) ^ 1, waits);
                    if (!ok) break;
                    prefill::tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < D; c += 16) {
                        float o[16];
                        unsigned int raw[16];
                        prefill::tmem_load16(outputs + c, o);
#pragma unroll
                        for (int i = 0; i < 16; ++i) raw[i] = __float_as_uint(o[i] * factor);
                        tmem_store16(outputs + c, raw);
                    }
                    tmem_wait_store();
                }
                if (step < turns) {
                    ok = wait_warp(&ctl->turn[tile][warp & 3], turn & 1, waits);
                    if (!ok) break;
                    ++turn;
                }
                // the maximum first, unscaled: what is left is small where a weight is not, whatever the maximum is
                const float base = m == -INFINITY ? 0.f : m;
                const unsigned long long multiplier2 = pair_of(multiplier, multiplier), base2 = pair_of(-base, -base);
                const unsigned long long shift2 = pair_of(kPromptShift<T>, kPromptShift<T>);
                unsigned long long sum0 = pair_of(0.f, 0.f), sum1 = sum0;
#pragma unroll
                for (int c = 0; c < kBlock; c += 32) {
                    unsigned int packed[16];
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        // the other tile's begin while the last of these are under way
                        if (c + i == kPassAt && step + tile < turns && lane == 0) mbar_arrive(&ctl->turn[tile ^ 1][warp & 3]);
                        const unsigned long long d0 = add_pair(pair_of(s[c + i], s[c + i + 1]), base2);
                        const unsigned long long d1 = add_pair(pair_of(s[c + i + 2], s[c + i + 3]), base2);
                        const unsigned long long e0 = fma_pair(d0, multiplier2, shift2), e1 = fma_pair(d1, multiplier2, shift2);
                        const float x0 = prefill::exp2_approx(pair_low(e0)), y0 = prefill::exp2_approx(pair_high(e0));
                        const float x1 = prefill::exp2_approx(pair_low(e1)), y1 = prefill::exp2_approx(pair_high(e1));
                        sum0 = add_pair(sum0, pair_of(x0, y0));
                        sum1 = add_pair(sum1, pair_of(x1, y1));
                        packed[i / 2] = pack_pair<T>(x0, y0);
                        packed[i / 2 + 1] = pack_pair<T>(x1, y1);
                    }
                    // weights of 32 keys take 16 columns, of scores that have been read
                    tmem_store16(scores + c / 2, packed);
                }
                tmem_wait_store();
                prefill::tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctl->p_full[slot]);
                sum0 = add_pair(sum0, sum1);
                l += pair_low(sum0) + pair_high(sum0);
            }
            info = (info + end - begin) % kInfos;
            // the outputs of the piece
            const bool any = first_block < blocks;
            if (any) {
                const int slot = tile * 2 + ((step - 1) & 1);
                ok = ok && wait_warp(&ctl->pv_done[slot], ((phase >> slot) & 1) ^ 1, waits);
                prefill::tc_fence_after();
            }
            float keep = 1.f, other = 0.f;   // factors of these outputs and of the other half's
            bool other_any = false;
            if (alone) {
                if (tile == 1) {
                    if (halves > 0) ok = ok && wait_warp(&ctl->half_taken, (halves - 1) & 1, waits);
                    ++halves;
                    ctl->half[r][0] = m;
                    ctl->half[r][1] = l;
                    prefill::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&ctl->half_ready);
                    release_work();
                    continue;
                }
                ok = ok && wait_warp(&ctl->half_ready, halves & 1, waits);
                ++halves;
                prefill::tc_fence_after();
                other_any = end - begin > 1;
                const float m1 = ctl->half[r][0], grown = fmaxf(m, m1), base = grown == -INFINITY ? 0.f : grown;
                keep = prefill::exp2_approx((m - base) * multiplier);
                other = prefill::exp2_approx((m1 - base) * multiplier);
                l = l * keep + ctl->half[r][1] * other;
                m = grown;
            }
            const bool whole = begin == 0 && end == u->blocks;
            const int unit_tokens = u->tokens;
            const int diagonal = max(begin, max(u->position, 0) / kBlock);   // the first block that a query may not see whole
            // Only of blocks whose products with values have been waited for: what is behind them is still being written.
            const int waited = alone ? end : blocks;
            bool any_odd = false;
            for (int b = diagonal; b < waited; ++b) any_odd |= ctl->odd[(info + 2 * kInfos - (end - b)) % kInfos] != 0;
            any_odd = __any_sync(0xffffffffu, any_odd);
            const float inverse = l == 0.f ? 0.f : 1.f / l;
            if (whole) keep *= inverse, other *= inverse;
            if (ok && any) {
                // a warp's 32 rows go through shared memory, 32 columns at a time, so that neighbouring lanes store
                // neighbouring 16 bytes of a row; the partial sums of a cut unit have an order of their own, rows first
                unsigned char* staging = stagings + warp * kStaging;
                float* partial = p.partial + static_cast<size_t>(blockIdx.x * 2 + (begin == 0 ? 1 : 0)) * kTiles * kRows * D +
                                 (tile * kRows + r) * 4;
                const size_t first_row = (static_cast<size_t>(u->first) + own * p.tile_tokens) * p.a.heads + u->head * group;
                const int tokens = min(unit_tokens - own * p.tile_tokens, p.tile_tokens);
                unsigned short* to = p.a.out + first_row * D + (lane & 3) * 8;
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    float o[32];
                    tmem_load32_async(outputs + c, o);
                    tmem_wait_load();
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] *= keep;
                    if (other_any) {
                        float o1[32];
                        tmem_load32_async(outputs + D + c, o1);
                        tmem_wait_load();
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = fmaf(o1[i], other, o[i]);
                    }
                    if (any_odd) {
                        float given[32];
#pragma unroll
                        for (int i = 0; i < 32; ++i) given[i] = o[i];
                        if (l != 0.f) give_back<T>(given, p.a, ctl, u, info, diagonal, waited, end, c, position);
                        __syncwarp();   // lanes come back at different times, and what follows is for all of them
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = given[i];
                    }
                    if (whole) {
#pragma unroll
                        for (int i = 0; i < 32; i += 8)   // 64 bytes a row, 16-byte pieces swizzled over eight rows
                            *reinterpret_cast<uint4*>(staging + lane * 64 + (((i >> 3) ^ ((lane >> 1) & 3)) << 4)) =
                                l == 0.f ? make_uint4(0u, 0u, 0u, 0u)
                                         : make_uint4(pack_pair<T>(o[i], o[i + 1]), pack_pair<T>(o[i + 2], o[i + 3]),
                                                      pack_pair<T>(o[i + 4], o[i + 5]), pack_pair<T>(o[i + 6], o[i + 7]));
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int at_row = i * 8 + (lane >> 2), row = r - lane + at_row;
                            const int row_token = row * group_inverse >> 16, in_group = row - row_token * group;
                            const uint4 v = *reinterpret_cast<const uint4*>(staging + at_row * 64 +
                                                                            (((lane & 3) ^ ((at_row >> 1) & 3)) << 4));
                            if (row_token < tokens)
                                *reinterpret_cast<uint4*>(to + (static_cast<size_t>(row_token) * p.a.heads + in_group) * D + c) =
                                    v;
                        }
                        __syncwarp();
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            *reinterpret_cast<float4*>(partial + static_cast<size_t>((c + i) / 4) * kTiles * kRows * 4) =
                                make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                    }
                }
            }
            if (!whole) {
                // Minus infinity says that nothing was written.  A maximum passes NaN by: where all scores of the piece are NaN
                // it is minus infinity too, and the sum says so.
                *reinterpret_cast<float2*>(
                    p.stats + (static_cast<size_t>(blockIdx.x * 2 + (begin == 0 ? 1 : 0)) * kTiles * kRows + tile * kRows + r) * 2) =
                    make_float2(any ? fmaxf(m * multiplier, -FLT_MAX) : -INFINITY, l);
                if (begin == 0) split = {u->first, u->head, u->tokens, u->pieces};
            }
            prefill::tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (any) mbar_arrive(&ctl->o_empty[tile]);
                if (other_any) mbar_arrive(&ctl->o_empty[1]);
                if (alone) mbar_arrive(&ctl->half_taken);
            }
            release_work();
        }
        if (tid == 0 && p.splits != nullptr)
            *reinterpret_cast<int4*>(p.splits + blockIdx.x) = make_int4(split.first, split.head, split.tokens, split.pieces);
        if (p.a.zero_rest != 0) {   // queries of no request: before the first one and behind the last one
            const size_t row = static_cast<size_t>(p.a.heads) * D / 8;
            const Request last = requests[p.a.requests - 1];
            const size_t front = requests[0].first * row, back = (last.first + last.tokens) * row;
            const size_t all = front + p.a.tokens * row - back;
            uint4* to = reinterpret_cast<uint4*>(p.a.out);
            for (size_t i = blockIdx.x * kTiles * 128 + tid; i < all; i += gridDim.x * kTiles * 128)
                to[i < front ? i : i - front + back] = make_uint4(0u, 0u, 0u, 0u);
        }
    }
    if (!ok && lane == 0) {
        waits->abort_flag = 1;
        if (p.a.status != nullptr) *p.a.status = MB_ST_PIPE_TIMEOUT;
    }
    prefill::tc_fence_before();
    __syncthreads();
    if (waits->abort_flag != 0) {   // copies and products that are under way end before the memory goes
        const unsigned long long start = global_timer_ns();
        while (global_timer_ns() - start < 200000ull) __nanosleep(1000);
        __syncthreads();
    }
    if (warp == 11) prefill::tmem_dealloc(tmem, kTmemColumns);
}

// The pieces of a unit that several CTAs share, in the order of its keys.  A thread has one row and D / 64 groups of four
// columns.  Latency bounds it, trips to L2 of about 800 cycles: the first two pieces are read before it is known whether a
// unit was cut here, statistics of all pieces at once, and sums of four pieces at a time (with two 16 tokens after 9,000,
// 18 pieces a unit, take 27.3 us instead of 25.8, with six 26.1, where 8 x 40 after 700 take 26.7, not 25.6).  One piece
// after the other it took 509 tokens after 16,000, 8/1 heads of 256, from 84 to 95 us.
constexpr int kJoinThreads = 128;
constexpr int kJoinRows = 8;

template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) prompt_join_kernel(const __grid_constant__ PromptArgs p) {
    extern __shared__ float2 statistics[];   // [pieces][kJoinRows]
    constexpr int kUnitRows = Config<D>::kTiles * kRows, kGroups = D / 64, kAhead = D == 256 ? 2 : 4;
    constexpr int kGroupColumns = kJoinThreads / kJoinRows * 4;
    static_assert(kGroups * kGroupColumns == D, "a thread has a group of columns of every kGroupColumns");
    const int group = p.a.heads / p.a.kv_heads;
    const int row = threadIdx.x % kJoinRows, r = blockIdx.y * kJoinRows + row, c = threadIdx.x / kJoinRows * 4;
    const int tile = r / kRows, in_tile = r % kRows, token = in_tile / group, mine = tile * p.tile_tokens + token;
    auto rows_of = [&](int i) {   // where the rows of piece i begin, among those of all pieces
        return ((static_cast<size_t>(blockIdx.x) + i) * 2 + (i == 0 ? 1 : 0)) * kUnitRows;
    };
    const float2* stats = reinterpret_cast<const float2*>(p.stats) + r;
    const float4* partial = reinterpret_cast<const float4*>(p.partial) + c / 4 * kUnitRows + r;
    float4 v[kAhead][kGroups];
    auto load = [&](int i, int q) {
#pragma unroll
        for (int g = 0; g < kGroups; ++g)
            v[i][g] = __ldcg(partial + rows_of(q) * (D / 4) + g * (kGroupColumns / 4) * kUnitRows);
    };
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int4 raw = __ldcg(reinterpret_cast<const int4*>(p.splits + blockIdx.x));
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (blockIdx.x + i < gridDim.x && token < p.tile_tokens) load(i, i);
    const Split split = {raw.x, raw.y, raw.z, raw.w};
    if (split.pieces == 0) return;
    for (int q = threadIdx.x / kJoinRows; q < split.pieces; q += kJoinThreads / kJoinRows)
        statistics[q * kJoinRows + row] = __ldcg(stats + rows_of(q));
    const bool counts = token < p.tile_tokens && mine < split.tokens;
    if (counts) {
#pragma unroll
        for (int i = 2; i < kAhead; ++i)
            if (i < split.pieces) load(i, i);
    }
    __syncthreads();
    if (!counts) return;
    float highest = -INFINITY;
    for (int q = 0; q < split.pieces; ++q) highest = fmaxf(highest, statistics[q * kJoinRows + row].x);
    float total = 0.f;
    float4 sum[kGroups];
#pragma unroll
    for (int g = 0; g < kGroups; ++g) sum[g] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int q0 = 0;;) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (q0 + i >= split.pieces) break;
            const float2 of = statistics[(q0 + i) * kJoinRows + row];
            if (of.x == -INFINITY) continue;   // nothing of it was written
            const float w = prefill::exp2_approx(of.x - highest);
            total = fmaf(w, of.y, total);
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                sum[g].x = fmaf(w, v[i][g].x, sum[g].x);
                sum[g].y = fmaf(w, v[i][g].y, sum[g].y);
                sum[g].z = fmaf(w, v[i][g].z, sum[g].z);
                sum[g].w = fmaf(w, v[i][g].w, sum[g].w);
            }
        }
        q0 += kAhead;
        if (q0 >= split.pieces) break;
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (q0 + i < split.pieces) load(i, q0 + i);
    }
    unsigned short* out =
        p.a.out + (static_cast<size_t>(split.first + mine) * p.a.heads + split.head * group + in_tile % group) * D + c;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) store_output<T>(out + g * kGroupColumns, sum[g], total);
}

// ---------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------
struct Shape {
    int tiles, tile_tokens, ctas, ring, smem;
    size_t stats, splits, bytes;   // workspace: partial sums, then from `stats` on the statistics, then the splits
    bool joined;
};

template <int D>
Shape shape_of(const AttentionArgs& a, int sms) {
    using C = Config<D>;
    Shape s;
    const int group = a.heads / a.kv_heads;
    s.tiles = C::kTiles;
    s.tile_tokens = kRows / group;
    // at most so many units, none longer than a row of the table
    const long long units = (a.tokens / (s.tile_tokens * s.tiles) + std::min(a.requests, a.tokens)) * static_cast<long long>(a.kv_heads);
    const long long capacity = static_cast<long long>(a.width) << a.page_shift;
    s.joined = capacity > kWholeKeys;
    const long long most = s.joined ? (units * (capacity + tile_cost(D)) + kLeastKeys - 1) / kLeastKeys : units;
    s.ctas = static_cast<int>(std::min<long long>(most, sms));
    const int rest = C::kTiles * (C::kQueryBytes + 4 * kStaging) + static_cast<int>(sizeof(PromptControl)) + 8 * (a.requests + 1) +
                     static_cast<int>(sizeof(Request)) * a.requests;
    s.ring = (kSmemLimit - rest) / C::kTileBytes;
    if (s.ring > kMaxTiles) s.ring = kMaxTiles;
    s.smem = rest + s.ring * C::kTileBytes;
    const size_t rows = static_cast<size_t>(s.ctas) * 2 * C::kTiles * kRows;
    s.stats = rows * D * 4;
    s.splits = s.stats + rows * 8;
    s.bytes = s.joined ? s.splits + s.ctas * sizeof(Split) : 0;
    return s;
}

Shape shape_of(const AttentionArgs& a, int sms) {
    return a.head_dim == 64 ? shape_of<64>(a, sms) : a.head_dim == 128 ? shape_of<128>(a, sms) : shape_of<256>(a, sms);
}

template <typename T, int D>
cudaError_t launch_prompt(const CUtensorMap& queries, const CUtensorMap& keys, const CUtensorMap& values,
                          const PromptArgs& args, const Shape& s, int device, cudaStream_t stream) {
    static std::atomic<unsigned long long> configured{0};   // devices, by their bits
    if (device >= 64 || !(configured.load(std::memory_order_relaxed) >> device & 1)) {
        const cudaError_t err = cudaFuncSetAttribute(prompt_attention_kernel<T, D>,
                                                     cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit);
        if (err != cudaSuccess) return err;
        if (device < 64) configured.fetch_or(1ull << device, std::memory_order_relaxed);
    }
    cudaError_t err = launch_early(prompt_attention_kernel<T, D>, dim3(s.ctas), kThreads, s.smem, 1, stream, queries, keys,
                                   values, args);
    if (err == cudaSuccess && s.joined)
        err = launch_early(prompt_join_kernel<T, D>, dim3(s.ctas, Config<D>::kTiles * kRows / kJoinRows), kJoinThreads,
                           s.ctas * kJoinRows * static_cast<int>(sizeof(float2)), 1, stream, args);
    return err;
}

template <typename T>
cudaError_t launch_prompt(const CUtensorMap& queries, const CUtensorMap& keys, const CUtensorMap& values,
                          const PromptArgs& args, const Shape& s, int device, cudaStream_t stream) {
    if (args.a.head_dim == 64) return launch_prompt<T, 64>(queries, keys, values, args, s, device, stream);
    if (args.a.head_dim == 128) return launch_prompt<T, 128>(queries, keys, values, args, s, device, stream);
    return launch_prompt<T, 256>(queries, keys, values, args, s, device, stream);
}

CUtensorMapDataType data_type(int element) {
    return element == MB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

// Boxes of one 128-byte column of up to a block of tokens of a page and head.
bool make_column_map(CUtensorMap* map, const AttentionArgs& a, const void* base, const Strides3& s, int element) {
    prefill::EncodeTiledFn fn = prefill::encode_tiled();
    if (fn == nullptr) return false;
    const int page = 1 << a.page_shift;
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(a.head_dim), static_cast<cuuint64_t>(page),
                                static_cast<cuuint64_t>(a.kv_heads), static_cast<cuuint64_t>(a.pages)};
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(s.token) * 2, static_cast<cuuint64_t>(s.head) * 2,
                                   static_cast<cuuint64_t>(s.page) * 2};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(page < kBlock ? page : kBlock), 1, 1};
    const cuuint32_t steps[4] = {1, 1, 1, 1};
    return fn(map, data_type(element), 4, const_cast<void*>(base), dims, strides, box, steps,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Boxes of one 128-byte column of the query heads of a key head, for the tokens of a tile.
bool make_query_map(CUtensorMap* map, const AttentionArgs& a, int element, int tile_tokens) {
    prefill::EncodeTiledFn fn = prefill::encode_tiled();
    if (fn == nullptr) return false;
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(a.head_dim), static_cast<cuuint64_t>(a.heads),
                                static_cast<cuuint64_t>(a.tokens)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(a.q.head) * 2, static_cast<cuuint64_t>(a.q.token) * 2};
    const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(a.heads / a.kv_heads), static_cast<cuuint32_t>(tile_tokens)};
    const cuuint32_t steps[3] = {1, 1, 1};
    return fn(map, data_type(element), 3, const_cast<unsigned short*>(a.query), dims, strides, box, steps,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

int prompt_admitted(const AttentionArgs& a) { return a.heads / a.kv_heads <= kRows ? MB_OK : MB_ERR_UNSUPPORTED; }

int64_t prompt_workspace(const AttentionArgs& a) {
    int device;
    cudaError_t err;
    const int sms = multiprocessors(&device, &err);
    if (err != cudaSuccess) return -cuda_error(err, "mb_paged_prefill_workspace");
    return static_cast<int64_t>(shape_of(a, sms).bytes);
}

int prompt_attention(const AttentionArgs& a, int element, void* workspace, cudaStream_t stream) {
    int device;
    cudaError_t err;
    const int sms = multiprocessors(&device, &err);
    if (err != cudaSuccess) return cuda_error(err, "mb_paged_prefill");
    const Shape s = shape_of(a, sms);
    if (s.ring < 3) return MB_ERR_RESOURCE;
    if (s.bytes != 0 && (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 256)) return MB_ERR_INVALID;
    CUtensorMap queries, keys, values;
    if (!make_query_map(&queries, a, element, s.tile_tokens) ||
        !make_column_map(&keys, a, a.key_pages, a.kpool, element) ||
        !make_column_map(&values, a, a.value_pages, a.vpool, element))
        return MB_ERR_UNSUPPORTED;
    PromptArgs args;
    args.a = a;
    args.tile_tokens = s.tile_tokens;
    args.ring = s.ring;
    args.scale_log2 = a.scale * kLog2e;
    char* base = static_cast<char*>(workspace);
    args.partial = reinterpret_cast<float*>(base);
    args.stats = reinterpret_cast<float*>(base + s.stats);
    args.splits = s.joined ? reinterpret_cast<Split*>(base + s.splits) : nullptr;
    err = element == MB_BF16 ? launch_prompt<__nv_bfloat16>(queries, keys, values, args, s, device, stream)
                             : launch_prompt<__half>(queries, keys, values, args, s, device, stream);
    return err == cudaSuccess ? MB_OK : cuda_error(err, "mb_paged_prefill");
}

}  // namespace paged
}  // namespace mb
