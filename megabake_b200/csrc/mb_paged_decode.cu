// Attention of one new token a request over a paged key-value cache (mb_paged_attention).
//
//   o = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m),   s_j = log2(e) scale q . k_j,   m = max_j s_j
//
// in one pass over the keys: a warp keeps a running m, sum and o of its own, and what it has is multiplied by
// 2^(m - m') when m grows to m'.  Every key and value is read once and used for at most a handful of queries
// (those of its head group), so HBM bounds it: 2 * 2 * kv_heads * head_dim bytes a key.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "mb_device.cuh"
#include "mb_kernels.h"
#include "mb_paged.cuh"
#include "mb_tensor.cuh"

namespace mb {
namespace paged {
namespace {

constexpr int kBlock = 64;          // keys of a ring stage
// Warps that compute, 16 keys of a stage each: two teams of four on stages in turn for 64-wide heads, whose stages are
// half as many bytes and take a team nearly as long (37 ragged contexts of up to 4,099 keys in pages of 16, 2 key heads:
// 22.0 -> 20.5 us).  The ring then has an even number of stages, so that a stage always belongs to one team, which sees
// every phase of its barrier: one that saw every other phase could not tell them apart by their parity.
template <int D>
constexpr int kTeams = D == 64 ? 2 : 1;
template <int D>
constexpr int kWarps = 4 * kTeams<D>;
template <int D>
constexpr int kThreads = 32 * (kWarps<D> + 1);
constexpr int kMaxStages = 16;
constexpr int kSmemLimit = 227 * 1024;
constexpr int kConsumerBarrier = 1;
// Of a run, where units are cut (one of 2,048 keys, 9/3 heads of 64: 7.4 us; 1: 7.7, 4: 8.0).
constexpr int kLeastBlocks = 2;
// Rows of the table that hold no more are not cut, whatever lengths are, which the host does not know: one launch and no
// scratch (33 keys: 4.5 us on the device in a table of 4 pages of 64, 7.2 to 7.6 in one of 128), and a CTA has eight blocks
// within about the time that joining pieces takes.
constexpr int kWholeBlocks = 8;

// What a CTA leaves behind about the unit that it began and others finish.
struct Split {
    int token, unit, pieces, unused;
};

struct DecodeArgs {
    AttentionArgs a;
    int subgroups;         // of a key head's queries: 8 or 16 each
    int stages;
    float scale_log2;
    Split* splits;         // [ctas]
    float* stats;          // [ctas][2][rows][2]: maximum, sum
    float* partial;        // [ctas][2][rows][D]
};

struct Control4 {
    unsigned long long full[kMaxStages], empty[kMaxStages], mask[kMaxStages];
    float2 stats[8][16];   // of every warp and query: maximum, sum
    int warp_sums[9];
    int abort_flag;
};

// ---------------------------------------------------------------------------------------
// The deal: blocks of 64 keys of all units (a token, a key head, 8 or 16 of its queries), one unit after the other,
// in equal runs over the CTAs.  A run begins and ends anywhere in a unit, so that contexts of any mix of
// lengths keep every SM busy until the end; at most the first and the last piece of a run are not whole.
// ---------------------------------------------------------------------------------------
struct Deal {
    const int* first_block;   // [tokens + 1] blocks (of one unit) before the token
    int tokens, units;        // units of a token
    long long total, per;
};

struct Piece {
    int token, unit, begin, end, blocks;   // blocks: of the whole unit
};

__device__ __forceinline__ Piece piece_at(const Deal& d, long long at, long long run_end) {
    int low = 0, high = d.tokens;   // first_block[low] * units <= at < first_block[high] * units
    while (high - low > 1) {
        const int middle = (low + high) >> 1;
        if (static_cast<long long>(d.first_block[middle]) * d.units <= at)
            low = middle;
        else
            high = middle;
    }
    Piece p;
    p.token = low;
    p.blocks = d.first_block[low + 1] - d.first_block[low];
    const long long rest = at - static_cast<long long>(d.first_block[low]) * d.units;
    // (a division of 64-bit numbers takes several hundred cycles)
    p.unit = rest >> 32 == 0 ? static_cast<int>(static_cast<unsigned int>(rest) / static_cast<unsigned int>(p.blocks))
                             : static_cast<int>(rest / p.blocks);
    p.begin = static_cast<int>(rest - static_cast<long long>(p.unit) * p.blocks);
    p.end = static_cast<int>(min(static_cast<long long>(p.blocks), p.begin + (run_end - at)));
    return p;
}

// The piece after `p`, which ended with its unit at `at`.
__device__ __forceinline__ void next_piece(const Deal& d, Piece& p, long long at, long long run_end) {
    if (++p.unit == d.units) {
        p.unit = 0;
        do ++p.token;
        while (d.first_block[p.token + 1] == d.first_block[p.token]);   // there is one with keys: `at` is before the end
        p.blocks = d.first_block[p.token + 1] - d.first_block[p.token];
    }
    p.begin = 0;
    p.end = static_cast<int>(min(static_cast<long long>(p.blocks), run_end - at));
}

// The first end or begin of a unit from `at` on.
__device__ __forceinline__ long long unit_boundary(const Deal& d, long long at) {
    if (at >= d.total) return at;
    const Piece p = piece_at(d, at, d.total);
    return p.begin == 0 ? at : at + p.blocks - p.begin;
}

__device__ __forceinline__ unsigned int movmatrix(unsigned int v) {
    unsigned int r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const unsigned int (&a)[4], unsigned int b0, unsigned int b1);
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&d)[4], const unsigned int (&a)[4], unsigned int b0,
                                                   unsigned int b1) {
    mma_bf16_16816(d, a[0], a[1], a[2], a[3], b0, b1);
}
template <>
__device__ __forceinline__ void mma<__half>(float (&d)[4], const unsigned int (&a)[4], unsigned int b0,
                                            unsigned int b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
        "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A weight as the sum of two 16-bit numbers, neither negative: the first is cut off, what that leaves out is less than a step
// of it, and the second keeps that to half a step of its own, so the product with the values sees weights of 16 (bf16) or
// 22 bits.  One 16-bit number would put as much error into the output as rounding the output does; the second product costs
// nothing here, where the matrix units wait for HBM.
//
// Both parts meet the same values, and an infinity times zero, or two of opposite signs, would be NaN.  So the second is at
// least the smallest number that counts, 2^-126 or 2^-24 beside weights of up to 2^-31 or 2^15, wherever the first is not zero.
template <typename T>
__device__ __forceinline__ void split_pair(float x, float y, unsigned int& high, unsigned int& low);
__device__ __forceinline__ unsigned int at_least_where(unsigned int v, unsigned int least, unsigned int where) {
    unsigned int r;
    asm("{\n\t.reg .b32 t;\n\t"
        "min.u16x2 t, %2, %3;\n\t"
        "max.u16x2 %0, %1, t;\n\t}"
        : "=r"(r)
        : "r"(v), "r"(least), "r"(where));
    return r;
}
template <>
__device__ __forceinline__ void split_pair<__nv_bfloat16>(float x, float y, unsigned int& high, unsigned int& low) {
    asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(high) : "f"(y), "f"(x));
    low = at_least_where(prefill::pack_bf16_pair(x - lo_bf16(high), y - hi_bf16(high)), 0x00800080u, high);
}
template <>
__device__ __forceinline__ void split_pair<__half>(float x, float y, unsigned int& high, unsigned int& low) {
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(high) : "f"(y), "f"(x));
    const __half2 h = *reinterpret_cast<const __half2*>(&high);
    const __half2 l = __floats2half2_rn(x - __low2float(h), y - __high2float(h));
    low = at_least_where(*reinterpret_cast<const unsigned int*>(&l), 0x00010001u, high);
}

__device__ __forceinline__ void tma_load_page(void* dst, const CUtensorMap* map, int place, int head, int page,
                                              unsigned long long* bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(smem_u32(dst)),
        "l"(map), "r"(0), "r"(place), "r"(0), "r"(head), "r"(page), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ float shuffled_max(float v) {
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
    return v;
}
__device__ __forceinline__ float shuffled_sum(float v) {
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

// A maximum that may be subtracted: of no keys at all it is minus infinity.
__device__ __forceinline__ float finite_base(float m) { return m == -INFINITY ? 0.f : m; }

// ---------------------------------------------------------------------------------------
// The kernel: one CTA per SM.  A warp copies pages into a ring of stages of 64 keys and their values; teams of four warps
// take stages in turn, a warp 16 of its keys.  Keys are the 16 rows of m16n8k16 products and queries its 8 columns, so that 8
// query heads of a key head cost what one costs; the scores come out with a query's keys spread over lanes, a transpose
// of 8 x 8 (movmatrix) makes them the second product's columns, and values are read transposed (ldmatrix.trans) as its
// rows: o^T = v^T p^T, whose columns are queries again, so that rescaling is by the lane's own two queries.
//
// Measured (us; floor at the measured copy bandwidth): 64 requests of 8,192 keys, 32/8 heads of 128: 313 to 348, by run (328),
// 6.2 to 6.9 TB/s, a few percent of it from L2 where passes follow one another; one of 131,071: 89 to 92 (82); 37 ragged ones
// of up to 4,099, 14/2 heads of 64, pages of 16: 20 (6), of which about 9 stream
// and the rest is latency: 4,400 cycles until the first keys are asked for and 1,700 until they are there, two merges of
// 2,000, the joining launch; one of 33 keys: 4.5.  Boxes issued by one lane, with 64-bit division for their places, instead
// of a box a lane and 32-bit: 24.0 us for the ragged ones, then 22.0.
// ---------------------------------------------------------------------------------------
template <typename T, int D, int N>   // N: 8-query columns of a unit
__global__ void __launch_bounds__(kThreads<D>, 1)
decode_attention_kernel(const __grid_constant__ CUtensorMap key_map, const __grid_constant__ CUtensorMap value_map,
                        const __grid_constant__ DecodeArgs p) {
    constexpr int kTeams = paged::kTeams<D>, kWarps = paged::kWarps<D>, kThreads = paged::kThreads<D>;
    constexpr int kTile = kBlock * D * 2;           // bytes of a stage's keys, and of its values
    constexpr int kQueries = 8 * N;
    constexpr int kMergeRow = D + 4;                // floats; the padding keeps a warp's stores off each other's banks
    extern __shared__ __align__(1024) unsigned char smem[];
    unsigned char* ring = smem;
    float* merge = reinterpret_cast<float*>(ring + static_cast<size_t>(p.stages) * 2 * kTile);  // [warps][queries][row]
    Control4* ctl = reinterpret_cast<Control4*>(merge + kWarps * kQueries * kMergeRow);
    int* first_block = reinterpret_cast<int*>(ctl + 1);                      // [tokens + 1]
    int* lengths = first_block + p.a.tokens + 1;                             // [tokens]
    int* table_rows = lengths + p.a.tokens;                                  // [tokens]

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int shift = p.a.page_shift, page = 1 << shift;
    if (tid == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(&ctl->full[s], 1);
            mbar_init(&ctl->empty[s], 4);
        }
        ctl->abort_flag = 0;
        mbar_init_fence();
    }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");

    // blocks before every token
    {
        const int each = (p.a.tokens + kThreads - 1) / kThreads;
        const int t0 = min(tid * each, p.a.tokens), t1 = min(t0 + each, p.a.tokens);
        const int capacity = p.a.width << shift;
        int sum = 0;
        for (int t = t0; t < t1; ++t) {
            const int r = p.a.index != nullptr ? p.a.index[t] : t;
            const int n = r >= 0 && r < p.a.requests ? min(max(p.a.lengths[r], 0), capacity) : 0;
            lengths[t] = n;
            table_rows[t] = r;
            sum += (n + kBlock - 1) / kBlock;
        }
        int inclusive = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int other = __shfl_up_sync(0xffffffffu, inclusive, d);
            if (lane >= d) inclusive += other;
        }
        if (lane == 31) ctl->warp_sums[warp] = inclusive;
        __syncthreads();
        int before = inclusive - sum;
        for (int w = 0; w < warp; ++w) before += ctl->warp_sums[w];
        for (int t = t0; t < t1; ++t) {
            first_block[t] = before;
            before += (lengths[t] + kBlock - 1) / kBlock;
        }
        if (t0 < p.a.tokens && t1 == p.a.tokens) first_block[p.a.tokens] = before;
        __syncthreads();
    }
    const int group = p.a.heads / p.a.kv_heads;
    Deal deal;
    deal.first_block = first_block;
    deal.tokens = p.a.tokens;
    deal.units = p.a.kv_heads * p.subgroups;
    deal.total = static_cast<long long>(first_block[p.a.tokens]) * deal.units;
    deal.per = deal.total >> 31 == 0 ? (static_cast<unsigned int>(deal.total) + gridDim.x - 1) / gridDim.x
                                     : (deal.total + gridDim.x - 1) / gridDim.x;
    deal.per = max(deal.per, p.splits != nullptr ? static_cast<long long>(kLeastBlocks) : 1);
    long long run_begin = min(blockIdx.x * deal.per, deal.total);
    long long run_end = min(run_begin + deal.per, deal.total);
    if (p.splits == nullptr) {   // no unit is cut: runs go from unit to unit
        run_begin = unit_boundary(deal, run_begin);
        run_end = unit_boundary(deal, run_end);
    }

    auto wait_warp = [&](unsigned long long* bar, unsigned int parity) {   // all lanes come to the same result
        return __all_sync(0xffffffffu, mbar_test_wait(bar, parity) ||
                                           wait_within(bar, parity, &ctl->abort_flag, p.a.wait_limit_ns)) != 0;
    };
    if (warp == kWarps) {
        // ---- copies
        int stage = 0;
        unsigned int round = 0;
        bool ok = true;
        const int rows_shift = min(shift, 6), rows = 1 << rows_shift;
        const int per_shift = 6 - rows_shift, per_block = 1 << per_shift;   // table entries of a block
        const int batch = 32 >> per_shift;                                  // blocks whose entries the lanes hold
        Piece piece = {};
        for (long long at = run_begin; ok && at < run_end;) {
            if (at == run_begin)
                piece = piece_at(deal, at, run_end);
            else
                next_piece(deal, piece, at, run_end);
            at += piece.end - piece.begin;
            const int n = lengths[piece.token], head = p.subgroups == 1 ? piece.unit : piece.unit / p.subgroups;
            const int* entries = p.a.table + static_cast<size_t>(table_rows[piece.token]) * p.a.width;
            const int entries_end = (n + page - 1) >> shift;
            auto entry_of = [&](int block) {   // this lane's entry of the batch that starts at `block`
                const int b = block + (lane >> per_shift);
                const int e = shift < 6 ? (b << per_shift) + (lane & (per_block - 1)) : b >> (shift - 6);
                int id = b < piece.end && e < entries_end ? entries[e] : -1;
                return id >= 0 && id < p.a.pages ? id : -1;
            };
            int next = entry_of(piece.begin);
            for (int b = piece.begin; ok && b < piece.end;) {
                const int mine = next;
                next = entry_of(b + batch);
                for (int j = 0; j < batch && b < piece.end; ++j, ++b) {
                    if (round > 0 && !wait_warp(&ctl->empty[stage], (round - 1) & 1)) {
                        ok = false;
                        break;
                    }
                    unsigned char* keys = ring + static_cast<size_t>(stage) * 2 * kTile;
                    const int left = n - b * kBlock;
                    const int id = __shfl_sync(0xffffffffu, mine, (j << per_shift) + (lane & (per_block - 1)));
                    const unsigned int valid = __ballot_sync(0xffffffffu, id >= 0) & ((2u << (per_block - 1)) - 1);
                    // lanes 0 .. 7: of which eight keys are on a page
                    const unsigned int eights =
                        __ballot_sync(0xffffffffu, lane < 8 && ((valid >> (lane >> (rows_shift - 3))) & 1u));
                    if (elect_one()) {
                        unsigned long long mask = 0;   // a byte for every bit of `eights`
                        if (eights == 0xffu)
                            mask = ~0ull;
                        else
                            for (int i = 0; i < 8; ++i) mask |= ((eights >> i) & 1u) ? 0xffull << (8 * i) : 0ull;
                        if (left < kBlock) mask &= (1ull << left) - 1;
                        ctl->mask[stage] = mask;
                        mbar_arrive_expect_tx(&ctl->full[stage], __popc(valid) * 2 * rows * D * 2);
                    }
                    __syncwarp();
                    const int place = page > kBlock ? (b * kBlock) & (page - 1) : 0;
                    if (per_block == 1) {
                        if (id >= 0 && elect_one()) {
                            tma_load_page(keys, &key_map, place, head, id, &ctl->full[stage]);
                            tma_load_page(keys + kTile, &value_map, place, head, id, &ctl->full[stage]);
                        }
                    } else if (lane < 2 * per_block && id >= 0) {   // a box a lane: keys, then values
                        const bool second = lane >= per_block;
                        tma_load_page(keys + (second ? kTile : 0) + (lane & (per_block - 1)) * rows * D * 2,
                                      second ? &value_map : &key_map, place, head, id, &ctl->full[stage]);
                    }
                    __syncwarp();
                    if (++stage == p.stages) {
                        stage = 0;
                        ++round;
                    }
                }
            }
        }
        if (!ok && lane == 0) {
            ctl->abort_flag = 1;
            if (p.a.status != nullptr) *p.a.status = MB_ST_PIPE_TIMEOUT;
        }
    } else {
        // ---- products
        int stage = 0;
        unsigned int round = 0;
        bool ok = true;
        Split split = {0, 0, 0, 0};
        const int rows = min(page, kBlock);
        const int key0 = (warp & 3) * 16, team = warp >> 2;
        // where this lane's rows of the 16 x 16 fragments lie: keys (not transposed) and values (transposed)
        const int k_row = key0 + (lane & 7) + ((lane >> 3) & 1) * 8, k_half = lane >> 4;
        const int v_row = key0 + (lane & 7) + (lane >> 4) * 8, v_half = (lane >> 3) & 1;
        // a box holds its rows once per 128-byte column: [box][column][row in the box]
        const int k_base = (k_row / rows) * rows * D * 2 + (k_row % rows) * 128;
        const int v_base = (v_row / rows) * rows * D * 2 + (v_row % rows) * 128;
        const int column = rows * 128;
        int turn = 0;   // of the teams
        Piece piece = {};
        for (long long at = run_begin; at < run_end;) {
            if (at == run_begin)
                piece = piece_at(deal, at, run_end);
            else
                next_piece(deal, piece, at, run_end);
            at += piece.end - piece.begin;
            const int n = lengths[piece.token], head = p.subgroups == 1 ? piece.unit : piece.unit / p.subgroups;
            const int sub = piece.unit - head * p.subgroups;
            const int first_query = head * group + sub * kQueries;
            const int queries = min(group - sub * kQueries, kQueries);
            // queries as columns of the first product: two neighbouring values and those 8 further on a 16-wide step
            unsigned int q[N][D / 16][2];
#pragma unroll
            for (int c = 0; c < N; ++c) {
                const int mine = c * 8 + (lane >> 2);
                const unsigned short* source = p.a.query + piece.token * p.a.q.token +
                                               (first_query + mine) * p.a.q.head + (lane & 3) * 2;
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    q[c][k][0] = mine < queries ? *reinterpret_cast<const unsigned int*>(source + k * 16) : 0u;
                    q[c][k][1] = mine < queries ? *reinterpret_cast<const unsigned int*>(source + k * 16 + 8) : 0u;
                }
            }
            const bool mine_is_last = p.a.key != nullptr && piece.end == piece.blocks && (((n - 1) & 63) >> 4) == (warp & 3);
            uint4 new_key, new_value;
            if (mine_is_last && lane < D / 8) {
                new_key = *reinterpret_cast<const uint4*>(p.a.key + piece.token * p.a.k.token + head * p.a.k.head + lane * 8);
                new_value =
                    *reinterpret_cast<const uint4*>(p.a.value + piece.token * p.a.v.token + head * p.a.v.head + lane * 8);
            }
            float m[N][2], l[N][2], o[N][D / 16][4];
#pragma unroll
            for (int c = 0; c < N; ++c) {
                m[c][0] = m[c][1] = -INFINITY;
                l[c][0] = l[c][1] = 0.f;
#pragma unroll
                for (int i = 0; i < D / 16; ++i) o[c][i][0] = o[c][i][1] = o[c][i][2] = o[c][i][3] = 0.f;
            }
            for (int b = piece.begin; b < piece.end; ++b) {
                const bool mine = turn == team;
                if (++turn == kTeams) turn = 0;
                if (!mine) {
                    if (++stage == p.stages) {
                        stage = 0;
                        ++round;
                    }
                    continue;
                }
                ok = ok && wait_warp(&ctl->full[stage], round & 1);
                if (!ok) continue;   // the barriers below are for all warps
                unsigned char* keys = ring + static_cast<size_t>(stage) * 2 * kTile;
                unsigned char* values = keys + kTile;
                const unsigned int mask = static_cast<unsigned int>(ctl->mask[stage] >> key0) & 0xffffu;
                if (mine_is_last && b == piece.blocks - 1 && ((mask >> ((n - 1) & 15)) & 1u)) {
                    // the token's own key and value: into the tile, and into their place in the pools
                    const int row = (n - 1) & 63;
                    if (lane < D / 8) {
                        const int place = (row / rows) * rows * D * 2 + (lane >> 3) * column + (row % rows) * 128 +
                                          (((lane & 7) ^ (row & 7)) << 4);
                        *reinterpret_cast<uint4*>(keys + place) = new_key;
                        *reinterpret_cast<uint4*>(values + place) = new_value;
                        if (sub == 0) {
                            const long long id =
                                p.a.table[static_cast<size_t>(table_rows[piece.token]) * p.a.width + ((n - 1) >> shift)];
                            const int in_page = (n - 1) & (page - 1);
                            *reinterpret_cast<uint4*>(const_cast<unsigned short*>(p.a.key_pages) + id * p.a.kpool.page +
                                                      in_page * p.a.kpool.token + head * p.a.kpool.head + lane * 8) = new_key;
                            *reinterpret_cast<uint4*>(const_cast<unsigned short*>(p.a.value_pages) + id * p.a.vpool.page +
                                                      in_page * p.a.vpool.token + head * p.a.vpool.head + lane * 8) =
                                new_value;
                        }
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before a copy lands here again
                    __syncwarp();
                }
                if (mask != 0) {
                    float s[N][4];
#pragma unroll
                    for (int c = 0; c < N; ++c) s[c][0] = s[c][1] = s[c][2] = s[c][3] = 0.f;
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        unsigned int a[4];
                        const int chunk = (k & 3) * 2 + k_half;
                        prefill::ldmatrix_x4(a, keys + k_base + (k >> 2) * column + ((chunk ^ (k_row & 7)) << 4));
#pragma unroll
                        for (int c = 0; c < N; ++c) mma<T>(s[c], a, q[c][k][0], q[c][k][1]);
                    }
                    const bool low_key = (mask >> (lane >> 2)) & 1u, high_key = (mask >> (8 + (lane >> 2))) & 1u;
                    unsigned int w[N][2][2];   // [high, low part][keys 0-7, 8-15]
#pragma unroll
                    for (int c = 0; c < N; ++c) {
                        s[c][0] = low_key ? s[c][0] * p.scale_log2 : -INFINITY;
                        s[c][1] = low_key ? s[c][1] * p.scale_log2 : -INFINITY;
                        s[c][2] = high_key ? s[c][2] * p.scale_log2 : -INFINITY;
                        s[c][3] = high_key ? s[c][3] * p.scale_log2 : -INFINITY;
                        float highest[2];
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            highest[i] = fmaxf(m[c][i], shuffled_max(fmaxf(s[c][i], s[c][i + 2])));
                        if (__any_sync(0xffffffffu, highest[0] != m[c][0] || highest[1] != m[c][1])) {
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                const float before = prefill::exp2_approx(m[c][i] - finite_base(highest[i]));
                                m[c][i] = highest[i];
                                l[c][i] *= before;
#pragma unroll
                                for (int t = 0; t < D / 16; ++t) {
                                    o[c][t][i] *= before;
                                    o[c][t][i + 2] *= before;
                                }
                            }
                        }
                        // the maximum first: a large one would swallow the shift
                        const float base0 = finite_base(m[c][0]), base1 = finite_base(m[c][1]);
                        s[c][0] = prefill::exp2_approx(s[c][0] - base0 + kWeightShift<T>);
                        s[c][1] = prefill::exp2_approx(s[c][1] - base1 + kWeightShift<T>);
                        s[c][2] = prefill::exp2_approx(s[c][2] - base0 + kWeightShift<T>);
                        s[c][3] = prefill::exp2_approx(s[c][3] - base1 + kWeightShift<T>);
                        l[c][0] += s[c][0] + s[c][2];
                        l[c][1] += s[c][1] + s[c][3];
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            unsigned int high, low;
                            split_pair<T>(s[c][2 * i], s[c][2 * i + 1], high, low);
                            w[c][0][i] = movmatrix(high);
                            w[c][1][i] = movmatrix(low);
                        }
                    }
                    // values of keys that do not count may be anything: 0 * NaN is NaN
                    const unsigned int near = mask >> ((lane & 3) * 2), far = near >> 8;
                    const unsigned int keep_near = ((near & 1u) ? 0xffffu : 0u) | ((near & 2u) ? 0xffff0000u : 0u);
                    const unsigned int keep_far = ((far & 1u) ? 0xffffu : 0u) | ((far & 2u) ? 0xffff0000u : 0u);
#pragma unroll
                    for (int t = 0; t < D / 16; ++t) {
                        unsigned int a[4];
                        const int chunk = (t & 3) * 2 + v_half;
                        prefill::ldmatrix_x4_trans(a, values + v_base + (t >> 2) * column + ((chunk ^ (v_row & 7)) << 4));
                        if (mask != 0xffffu) {
                            a[0] &= keep_near;
                            a[1] &= keep_near;
                            a[2] &= keep_far;
                            a[3] &= keep_far;
                        }
#pragma unroll
                        for (int c = 0; c < N; ++c) {
                            mma<T>(o[c][t], a, w[c][0][0], w[c][0][1]);
                            mma<T>(o[c][t], a, w[c][1][0], w[c][1][1]);
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctl->empty[stage]);
                if (++stage == p.stages) {
                    stage = 0;
                    ++round;
                }
            }
            // the warps' shares of the piece, every one relative to its own maximum
#pragma unroll
            for (int c = 0; c < N; ++c)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int mine = c * 8 + (lane & 3) * 2 + i;
                    l[c][i] = shuffled_sum(l[c][i]);
                    if (lane < 4) ctl->stats[warp][mine] = make_float2(m[c][i], l[c][i]);
                    if (mine < queries) {
                        float* to = merge + (warp * kQueries + mine) * kMergeRow + (lane >> 2);
#pragma unroll
                        for (int t = 0; t < D / 16; ++t) {
                            to[t * 16] = o[c][t][i];
                            to[t * 16 + 8] = o[c][t][i + 2];
                        }
                    }
                }
            named_barrier(kConsumerBarrier, kWarps * 32);
            const bool whole = piece.begin == 0 && piece.end == piece.blocks;
            const int slot = blockIdx.x * 2 + (piece.begin == 0 ? 1 : 0);
            for (int i = tid; i < queries * (D / 4); i += kWarps * 32) {
                const int mine = i / (D / 4), c = i % (D / 4) * 4;
                float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
                float highest = -INFINITY, total = 0.f;
                float2 share[kWarps];
#pragma unroll
                for (int other = 0; other < kWarps; ++other) {
                    share[other] = ctl->stats[other][mine];
                    highest = fmaxf(highest, share[other].x);
                }
#pragma unroll
                for (int other = 0; other < kWarps; ++other) {
                    const float4 v = *reinterpret_cast<const float4*>(merge + (other * kQueries + mine) * kMergeRow + c);
                    const float factor = prefill::exp2_approx(share[other].x - finite_base(highest));
                    total = fmaf(factor, share[other].y, total);
                    sum.x = fmaf(factor, v.x, sum.x);
                    sum.y = fmaf(factor, v.y, sum.y);
                    sum.z = fmaf(factor, v.z, sum.z);
                    sum.w = fmaf(factor, v.w, sum.w);
                }
                if (whole) {
                    store_output<T>(p.a.out + (static_cast<size_t>(piece.token) * p.a.heads + first_query + mine) * D + c,
                                    sum, total);
                } else {
                    *reinterpret_cast<float4*>(p.partial + (static_cast<size_t>(slot) * kQueries + mine) * D + c) = sum;
                    if (c == 0)
                        *reinterpret_cast<float2*>(p.stats + (static_cast<size_t>(slot) * kQueries + mine) * 2) =
                            make_float2(highest, total);
                }
            }
            if (!whole && piece.begin == 0) {
                const long long unit_end = at - piece.end + piece.blocks;
                split = {piece.token, piece.unit, static_cast<int>((unit_end - 1) / deal.per - blockIdx.x) + 1, 0};
            }
            named_barrier(kConsumerBarrier, kWarps * 32);   // the shares have been read
        }
        if (tid == 0 && p.splits != nullptr) *reinterpret_cast<int4*>(p.splits + blockIdx.x) = *reinterpret_cast<int4*>(&split);
        if (!ok && lane == 0) {
            ctl->abort_flag = 1;
            if (p.a.status != nullptr) *p.a.status = MB_ST_PIPE_TIMEOUT;
        }
        // tokens without a key
        for (int t = blockIdx.x; t < p.a.tokens; t += gridDim.x) {
            if (lengths[t] != 0) continue;
            uint4* to = reinterpret_cast<uint4*>(p.a.out + static_cast<size_t>(t) * p.a.heads * D);
            for (int i = tid; i < p.a.heads * D / 8; i += kWarps * 32) to[i] = make_uint4(0u, 0u, 0u, 0u);
        }
    }
    __syncthreads();
    if (ctl->abort_flag != 0) {   // copies that are under way land before the memory goes
        const unsigned long long start = global_timer_ns();
        while (global_timer_ns() - start < 200000ull) __nanosleep(1000);
    }
}

// The pieces of a unit that several CTAs share, in the order of its keys.  CTA (c, q): query q of the unit that CTA c of
// the kernel before began and did not finish, if there is one.
constexpr int kJoinThreads = 256;
constexpr int kJoinPieces = 1024;   // at most as many as CTAs

template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const __grid_constant__ DecodeArgs p, const int rows) {
    __shared__ float weight[kJoinPieces];
    __shared__ float4 sums[kJoinThreads];
    __shared__ float total_smem;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int4 raw = __ldcg(reinterpret_cast<const int4*>(p.splits + blockIdx.x));
    const int token = raw.x, unit = raw.y, pieces = raw.z;
    const int group = p.a.heads / p.a.kv_heads, mine = blockIdx.y;
    const int head = unit / p.subgroups, sub = unit % p.subgroups;
    if (pieces == 0 || mine >= group - sub * rows) return;
    auto slot_of = [&](int i) { return (static_cast<size_t>(blockIdx.x) + i) * 2 + (i == 0 ? 1 : 0); };
    const int tid = threadIdx.x;
    if (tid < 32) {
        float highest = -INFINITY;
        for (int i = tid; i < pieces; i += 32) {
            const float m = __ldcg(p.stats + (slot_of(i) * rows + mine) * 2);
            weight[i] = m;
            highest = fmaxf(highest, m);
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) highest = fmaxf(highest, __shfl_xor_sync(0xffffffffu, highest, d));
        float total = 0.f;
        for (int i = tid; i < pieces; i += 32) {
            weight[i] = prefill::exp2_approx(weight[i] - finite_base(highest));
            total += weight[i] * __ldcg(p.stats + (slot_of(i) * rows + mine) * 2 + 1);
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
        if (tid == 0) total_smem = total;
    }
    __syncthreads();
    constexpr int kColumns = D / 4, kGroups = kJoinThreads / kColumns;
    const int c = tid % kColumns, g = tid / kColumns;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = g; i < pieces; i += kGroups) {
        const float4 v = __ldcg(reinterpret_cast<const float4*>(p.partial + (slot_of(i) * rows + mine) * D) + c);
        const float w = weight[i];
        sum.x = fmaf(w, v.x, sum.x);
        sum.y = fmaf(w, v.y, sum.y);
        sum.z = fmaf(w, v.z, sum.z);
        sum.w = fmaf(w, v.w, sum.w);
    }
    sums[tid] = sum;
    __syncthreads();
    if (g != 0) return;
    for (int other = 1; other < kGroups; ++other) {
        const float4 v = sums[other * kColumns + c];
        sum.x += v.x;
        sum.y += v.y;
        sum.z += v.z;
        sum.w += v.w;
    }
    store_output<T>(p.a.out + (static_cast<size_t>(token) * p.a.heads + head * group + sub * rows + mine) * D + c * 4, sum,
                    total_smem);
}

// ---------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------
struct Shape {
    int columns, subgroups, rows, ctas, stages, smem;
    size_t splits, stats, bytes;   // workspace: partial sums, then from `stats` on the statistics, then the splits
    bool joined;
};

Shape shape_of(const AttentionArgs& a, int sms) {
    Shape s;
    const int group = a.heads / a.kv_heads;
    s.columns = group <= 8 ? 1 : 2;
    s.rows = 8 * s.columns;
    s.subgroups = (group + s.rows - 1) / s.rows;
    const int blocks = ((a.width << a.page_shift) + kBlock - 1) / kBlock;   // of a full row
    const long long most = static_cast<long long>(a.tokens) * a.kv_heads * s.subgroups * blocks;
    s.ctas = static_cast<int>(most < sms ? most : sms);
    s.joined = blocks > kWholeBlocks;
    const int tile = 2 * kBlock * a.head_dim * 2;
    const int teams = a.head_dim == 64 ? kTeams<64> : kTeams<128>, warps = 4 * teams;
    const int rest = warps * s.rows * (a.head_dim + 4) * 4 + static_cast<int>(sizeof(Control4)) + (3 * a.tokens + 1) * 4;
    s.stages = (kSmemLimit - rest) / tile;
    if (s.stages > kMaxStages) s.stages = kMaxStages;
    s.stages -= s.stages % teams;
    s.smem = s.stages * tile + rest;
    const size_t pieces = static_cast<size_t>(s.ctas) * 2 * s.rows;
    s.stats = pieces * a.head_dim * 4;
    s.splits = s.stats + pieces * 8;
    s.bytes = s.joined ? s.splits + s.ctas * sizeof(Split) : 0;
    return s;
}

template <typename T, int D>
cudaError_t launch_join(const DecodeArgs& args, const Shape& s, cudaStream_t stream) {
    const int group = args.a.heads / args.a.kv_heads;
    return launch_early(join_kernel<T, D>, dim3(s.ctas, group < s.rows ? group : s.rows), kJoinThreads, 0, 1, stream, args,
                        s.rows);
}

template <typename T, int D, int N>
cudaError_t launch_decode(const CUtensorMap& keys, const CUtensorMap& values, const DecodeArgs& args, const Shape& s,
                          int device, cudaStream_t stream) {
    static std::atomic<unsigned long long> configured{0};   // devices, by their bits
    if (device >= 64 || !(configured.load(std::memory_order_relaxed) >> device & 1)) {
        const cudaError_t err = cudaFuncSetAttribute(decode_attention_kernel<T, D, N>,
                                                     cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit);
        if (err != cudaSuccess) return err;
        if (device < 64) configured.fetch_or(1ull << device, std::memory_order_relaxed);
    }
    cudaError_t err = launch_early(decode_attention_kernel<T, D, N>, dim3(s.ctas), kThreads<D>, s.smem, 1, stream, keys, values,
                                   args);
    if (err == cudaSuccess && s.joined) err = launch_join<T, D>(args, s, stream);
    return err;
}

template <typename T>
cudaError_t launch_decode(const CUtensorMap& keys, const CUtensorMap& values, const DecodeArgs& args, const Shape& s,
                          int device, cudaStream_t stream) {
    if (args.a.head_dim == 64)
        return s.columns == 1 ? launch_decode<T, 64, 1>(keys, values, args, s, device, stream)
                              : launch_decode<T, 64, 2>(keys, values, args, s, device, stream);
    if (args.a.head_dim == 128)
        return s.columns == 1 ? launch_decode<T, 128, 1>(keys, values, args, s, device, stream)
                              : launch_decode<T, 128, 2>(keys, values, args, s, device, stream);
    return s.columns == 1 ? launch_decode<T, 256, 1>(keys, values, args, s, device, stream)
                          : launch_decode<T, 256, 2>(keys, values, args, s, device, stream);
}

}  // namespace

// Boxes of up to 64 tokens of a page and head, every row cut into 128-byte columns: [column][row], swizzled.
bool make_page_map(CUtensorMap* map, const AttentionArgs& a, const void* base, const Strides3& s, int element) {
    prefill::EncodeTiledFn fn = prefill::encode_tiled();
    if (fn == nullptr) return false;
    const int page = 1 << a.page_shift;
    const cuuint64_t dims[5] = {64, static_cast<cuuint64_t>(page), static_cast<cuuint64_t>(a.head_dim / 64),
                                static_cast<cuuint64_t>(a.kv_heads), static_cast<cuuint64_t>(a.pages)};
    const cuuint64_t strides[4] = {static_cast<cuuint64_t>(s.token) * 2, 128, static_cast<cuuint64_t>(s.head) * 2,
                                   static_cast<cuuint64_t>(s.page) * 2};
    const cuuint32_t box[5] = {64, static_cast<cuuint32_t>(page < kBlock ? page : kBlock),
                               static_cast<cuuint32_t>(a.head_dim / 64), 1, 1};
    const cuuint32_t steps[5] = {1, 1, 1, 1, 1};
    return fn(map, element == MB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5,
              const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int multiprocessors(int* device, cudaError_t* err) {
    static std::atomic<int> known[64];
    *err = cudaGetDevice(device);
    if (*err != cudaSuccess) return 0;
    int sms = *device < 64 ? known[*device].load(std::memory_order_relaxed) : 0;
    if (sms == 0) {
        *err = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, *device);
        if (*err != cudaSuccess) return 0;
        if (*device < 64) known[*device].store(sms, std::memory_order_relaxed);
    }
    return sms;
}

int decode_admitted(const AttentionArgs& a) {
    if (a.tokens > kMaxRows || (static_cast<long long>(a.width) << a.page_shift) * a.tokens >= 1ll << 37)
        return MB_ERR_UNSUPPORTED;
    return MB_OK;
}

int64_t decode_workspace(const AttentionArgs& a) {
    int device;
    cudaError_t err;
    const int sms = multiprocessors(&device, &err);
    if (err != cudaSuccess) return -cuda_error(err, "mb_paged_attention_workspace");
    return static_cast<int64_t>(shape_of(a, sms).bytes);
}

int decode_attention(const AttentionArgs& a, int element, void* workspace, cudaStream_t stream) {
    int device;
    cudaError_t err;
    const int sms = multiprocessors(&device, &err);
    if (err != cudaSuccess) return cuda_error(err, "mb_paged_attention");
    const Shape s = shape_of(a, sms);
    if (s.stages < 2) return MB_ERR_RESOURCE;
    if (s.bytes != 0 && (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 256)) return MB_ERR_INVALID;
    CUtensorMap keys, values;
    if (!make_page_map(&keys, a, a.key_pages, a.kpool, element) ||
        !make_page_map(&values, a, a.value_pages, a.vpool, element))
        return MB_ERR_UNSUPPORTED;
    DecodeArgs args;
    args.a = a;
    args.subgroups = s.subgroups;
    args.stages = s.stages;
    args.scale_log2 = a.scale * kLog2e;
    char* base = static_cast<char*>(workspace);
    args.partial = reinterpret_cast<float*>(base);
    args.stats = reinterpret_cast<float*>(base + s.stats);
    args.splits = s.joined ? reinterpret_cast<Split*>(base + s.splits) : nullptr;
    err = element == MB_BF16 ? launch_decode<__nv_bfloat16>(keys, values, args, s, device, stream)
                             : launch_decode<__half>(keys, values, args, s, device, stream);
    return err == cudaSuccess ? MB_OK : cuda_error(err, "mb_paged_attention");
}

}  // namespace paged
}  // namespace mb
