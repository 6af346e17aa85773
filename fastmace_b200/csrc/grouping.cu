// Rows by group: a stable counting sort of row numbers by a small key (the species of an atom, the expert of a row).
//
//   count:  a CTA counts the keys of kRowsPerCta consecutive rows
//   scan:   per group, the counts of the CTAs before each CTA, and the total
//   place:  every warp of a CTA owns consecutive rows; the warps' own counts give each its first place per group, and inside
//           32 rows the lanes with the same key find their order by votes; no atomics on results, so the order is the one of
//           the row numbers
//
// Rows whose key is no group come behind all groups. Up to kRowsPerCta rows `place` alone does it: one launch.
// Bound by latency: 8 bytes move per row and the second pass reads keys from L2. A lane asks for its keys all at once and keeps them for
// both passes of `place`; one at a time, each waited for, 1,944 rows took 14 us. A call: 1,944 rows by 2 keys 11 us (one launch of
// one CTA, of which the launch is most), 2,100,003 rows by 128 keys 35 us (three launches; 17 MB, 2.6 us of memory).

#include "early.cuh"

#include <algorithm>

namespace fmb {

namespace {

constexpr int kKeys = 8;                                  // per lane
constexpr int kRowsPerWarp = 32 * kKeys;
constexpr int kWarps = 32;                                // of a CTA that groups; of one that sorts tokens also kFewWarps
constexpr int kFewWarps = 8;
constexpr int kRowsPerCta = kWarps * kRowsPerWarp;

// A pass over some bits of keys that are too many for one table (sort_tokens): the row in place i is from[i], or i; a key that
// is no token counts as `vocabulary`, behind all others; the groups are the values of its bits from `shift` on.
struct Digit {
    const int32_t* from;
    int32_t* sorted_keys;                                 // of the last pass: the keys in their order
    int vocabulary, shift, mask;
};

// as kept: `groups` stands for "no group"
template <typename K>
__device__ __forceinline__ int group_of(K key, int groups) { return key < 0 || key >= (K)groups ? groups : (int)key; }

// the groups of this lane's rows begin + 32 i + lane, -1 for rows past the end
template <typename K, bool DIGIT>
__device__ __forceinline__ void load_keys(const K* __restrict__ keys, const Digit& d, long long begin, long long rows, int groups, int (&g)[kKeys]) {
    const int lane = threadIdx.x & 31;
    K key[kKeys];
    int at[kKeys];
    if (DIGIT && d.from) {
#pragma unroll
        for (int i = 0; i < kKeys; ++i) at[i] = begin + 32 * i + lane < rows ? d.from[begin + 32 * i + lane] : 0;
    }
#pragma unroll
    for (int i = 0; i < kKeys; ++i) {
        const long long row = begin + 32 * i + lane;
        key[i] = row < rows ? keys[DIGIT && d.from ? at[i] : row] : (K)-1;
    }
#pragma unroll
    for (int i = 0; i < kKeys; ++i)
        g[i] = begin + 32 * i + lane >= rows ? -1 : DIGIT ? group_of(key[i], d.vocabulary) >> d.shift & d.mask : group_of(key[i], groups);
}

// Lanes whose rows have this lane's group, for each of its rows, by a vote per bit of the group's number: 3 instructions a bit,
// where a match instruction holds the SM's one unit for 80 cycles (2.1 M rows: 19 us for the counts alone).
__device__ __forceinline__ void match_groups(const int (&g)[kKeys], int bits, unsigned (&same)[kKeys]) {
#pragma unroll
    for (int i = 0; i < kKeys; ++i) {
        const unsigned there = __ballot_sync(0xffffffffu, g[i] >= 0);
        same[i] = g[i] >= 0 ? there : 0;
    }
    for (int b = 0; b < bits; ++b) {
#pragma unroll
        for (int i = 0; i < kKeys; ++i) {
            const bool set = (g[i] >> b) & 1;
            const unsigned with = __ballot_sync(0xffffffffu, set);
            same[i] &= set ? with : ~with;
        }
    }
}

// of the 32 warps' counts of group g: what the warps before lane `w`'s have, and all of them (lane = warp)
__device__ __forceinline__ int warps_before(int mine, int& all) {
    const int lane = threadIdx.x & 31;
    int inclusive = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, inclusive, o);
        if (lane >= o) inclusive += up;
    }
    all = __shfl_sync(0xffffffffu, inclusive, 31);
    return inclusive - mine;
}

template <typename K, bool DIGIT, int WARPS>
__global__ void __launch_bounds__(32 * WARPS)
k_group_count(const K* keys, Digit d, long long rows, int groups, int32_t* __restrict__ table) {
    constexpr int kThreads = 32 * WARPS, kRowsPerCta = WARPS * kRowsPerWarp;
    __shared__ int counts[FMB_MAX_GROUPS + 1];
    const int width = groups + 1;
    if (DIGIT) {
        let_next_come();
        kernels_before(keys, d.from);
    }
    int g[kKeys];
    load_keys<K, DIGIT>(keys, d, (long long)blockIdx.x * kRowsPerCta + (threadIdx.x >> 5) * kRowsPerWarp, rows, groups, g);
    for (int q = threadIdx.x; q < width; q += kThreads) counts[q] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kKeys; ++i)
        if (g[i] >= 0) atomicAdd(counts + g[i], 1);               // sums of integers: the same in any order
    __syncthreads();
    for (int q = threadIdx.x; q < width; q += kThreads) table[(long long)blockIdx.x * width + q] = counts[q];
}

// table[cta][g] becomes the rows of g in the CTAs before; totals[g]. A CTA takes 32 groups, its 32 warps a share of the
// table's rows each.
template <bool DIGIT>
__global__ void __launch_bounds__(1024)
k_group_scan(int32_t* __restrict__ table, int32_t* __restrict__ totals, int ctas, int width) {
    if (DIGIT) {
        let_next_come();
        kernels_before(table);
    }
    __shared__ int part[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = blockIdx.x * 32 + lane;
    const int share = (ctas + 31) / 32, begin = warp * share, end = min(ctas, begin + share);
    int sum = 0;
    if (g < width) {
#pragma unroll 8
        for (int c = begin; c < end; ++c) sum += table[(long long)c * width + g];
    }
    part[warp][lane] = sum;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < warp; ++w) before += part[w][lane];
    if (g >= width) return;
    for (int c0 = begin; c0 < end; c0 += 8) {
        int here[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) here[i] = c0 + i < end ? table[(long long)(c0 + i) * width + g] : 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (c0 + i < end) table[(long long)(c0 + i) * width + g] = before;
            before += here[i];
        }
    }
    if (warp == 31) totals[g] = before;
}

// starts[g] = sum of starts[0 .. g) for g < width, by the whole CTA
template <int WARPS>
__device__ __forceinline__ void exclusive_starts(int* starts, int width) {
    constexpr int kThreads = 32 * WARPS;
    __shared__ int warp_total[WARPS];
    const int per = (width + kThreads - 1) / kThreads, begin = min(width, (int)threadIdx.x * per), end = min(width, begin + per);
    int sum = 0, all;
    for (int i = begin; i < end; ++i) sum += starts[i];
    int before = warps_before(sum, all);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (lane == 31) warp_total[warp] = all;
    __syncthreads();
    int ahead = lane < warp ? warp_total[lane] : 0;
    before += warp_sum(ahead);
    for (int i = begin; i < end; ++i) {
        const int here = starts[i];
        starts[i] = before;
        before += here;
    }
    __syncthreads();
}

// Distance of the warps' counts, odd: a warp reads one count of each (65,536 rows by the 512 values of nine bits: 32 us, and 9 so)
__host__ __device__ constexpr int place_stride(int width) { return width | 1; }
constexpr int place_smem(int width, int warps) { return (warps * place_stride(width) + 2 * width + warps * kRowsPerWarp) * 4; }

// ALONE: the only CTA, which takes its own counts for the totals. The CTA's rows are put in order in shared memory first, so
// that the rows of a group leave in one run.
template <typename K, bool ALONE, bool DIGIT, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, ALONE ? 1 : 64 / WARPS)
k_group_place(const K* keys, Digit d, long long rows, int groups, int bits, const int32_t* table, const int32_t* totals,
              int32_t* __restrict__ order, int32_t* __restrict__ offsets) {
    static_assert(!(ALONE && DIGIT), "rows of one CTA are ranked, not sorted by digits");
    constexpr int kThreads = 32 * WARPS, kRowsPerCta = WARPS * kRowsPerWarp;
    extern __shared__ int counts[];                       // [WARPS][stride], [groups + 1] starts of the CTA, [groups + 1] of all, rows
    const int width = groups + 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, stride = place_stride(width);
    int* const here = counts + WARPS * stride;
    int* const starts = ALONE ? here : here + width;
    int* const sorted = here + 2 * width;                 // row of the CTA | group << 13
    const long long first = (long long)blockIdx.x * kRowsPerCta;
    if (DIGIT) {
        let_next_come();
        kernels_before(keys, d.from, table, totals);
    }
    int g[kKeys], rank[kKeys];
    load_keys<K, DIGIT>(keys, d, first + warp * kRowsPerWarp, rows, groups, g);
    const int warps = ALONE ? (int)((rows + kRowsPerWarp - 1) / kRowsPerWarp) : WARPS;         // that have rows
    for (int i = threadIdx.x; i < warps * stride; i += kThreads) counts[i] = 0;
    if (!ALONE)
        for (int q = threadIdx.x; q < width; q += kThreads) starts[q] = totals[q];
    unsigned same[kKeys];
    match_groups(g, bits, same);
    __syncthreads();
    int* const mine = counts + warp * stride;
#pragma unroll
    for (int i = 0; i < kKeys; ++i) {
        const int before = g[i] >= 0 ? mine[g[i]] : 0, ahead = __popc(same[i] & ((1u << lane) - 1u));
        __syncwarp();
        if (g[i] >= 0 && ahead == 0) mine[g[i]] = before + __popc(same[i]);
        rank[i] = before + ahead;
        __syncwarp();
    }
    __syncthreads();
    if (DIGIT && width >= kThreads / 4) {
        // a thread per group, whose counts it reads one after the other (a warp for each waits 16 times for its shuffles at 512)
        for (int q = threadIdx.x; q < width; q += kThreads) {
            int all = 0;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const int count = counts[w * stride + q];
                counts[w * stride + q] = all;
                all += count;
            }
            here[q] = all;
        }
    } else {
        for (int q = warp; q < width; q += WARPS) {
            int all;
            const int before = warps_before(lane < warps ? counts[lane * stride + q] : 0, all);
            if (lane < warps) counts[lane * stride + q] = before;
            if (lane == 0) here[q] = all;
        }
    }
    __syncthreads();
    exclusive_starts<WARPS>(here, width);
    if (!ALONE) exclusive_starts<WARPS>(starts, width);
    if (!DIGIT && blockIdx.x == 0)
        for (int q = threadIdx.x; q < width; q += kThreads) offsets[q] = starts[q];
#pragma unroll
    for (int i = 0; i < kKeys; ++i)
        if (g[i] >= 0) sorted[here[g[i]] + mine[g[i]] + rank[i]] = (warp * kRowsPerWarp + 32 * i + lane) | g[i] << 13;
    __syncthreads();
    if (!ALONE) {
        // where the CTA's rows of a group go, less their place among its own
        for (int q = threadIdx.x; q < width; q += kThreads) starts[q] += table[(long long)blockIdx.x * width + q] - here[q];
        __syncthreads();
    }
    const int count = (int)min((long long)kRowsPerCta, rows - first);
    int32_t row[kKeys];
    int to[kKeys];
#pragma unroll
    for (int j = 0; j < kKeys; ++j) {
        const int i = threadIdx.x + j * kThreads, v = i < count ? sorted[i] : 0;
        to[j] = i < count ? (ALONE ? 0 : starts[v >> 13]) + i : -1;
        row[j] = (int32_t)(first + (v & (kRowsPerCta - 1)));
    }
    if (DIGIT && d.from) {
#pragma unroll
        for (int j = 0; j < kKeys; ++j)
            if (to[j] >= 0) row[j] = d.from[row[j]];
    }
#pragma unroll
    for (int j = 0; j < kKeys; ++j)
        if (to[j] >= 0) order[to[j]] = row[j];
    if (DIGIT && d.sorted_keys) {
        K key[kKeys];
#pragma unroll
        for (int j = 0; j < kKeys; ++j) key[j] = to[j] >= 0 ? keys[row[j]] : (K)0;
#pragma unroll
        for (int j = 0; j < kKeys; ++j)
            if (to[j] >= 0) d.sorted_keys[to[j]] = group_of(key[j], d.vocabulary);
    }
}

// one stable pass: counts, their sums over the CTAs, places; a launch alone where one CTA takes all rows. The passes of tokens, of which there
// are two and more behind them, come early.
template <typename K, bool DIGIT, int WARPS>
int sort_pass(const K* keys, const Digit& d, long long rows, int groups, int32_t* order, int32_t* offsets, int32_t* scratch, cudaStream_t stream) {
    const int width = groups + 1, ctas = ceil_div(rows, WARPS * kRowsPerWarp);
    const int smem = place_smem(width, WARPS), most = place_smem(FMB_MAX_GROUPS + 1, WARPS), bits = 32 - __builtin_clz(groups);
    auto launch = [&](auto kernel, int grid, int threads, int bytes, auto... arguments) -> cudaError_t {
        if constexpr (DIGIT) return launch_early(kernel, grid, threads, bytes, stream, arguments...);
        kernel<<<grid, threads, bytes, stream>>>(arguments...);
        return cudaGetLastError();
    };
    if constexpr (!DIGIT) {                      // (fewer tokens are ranked)
        if (ctas <= 1) {
            FMB_CUDA_CHECK(opt_in_shared_memory((const void*)k_group_place<K, true, false, WARPS>, most));
            k_group_place<K, true, false, WARPS><<<1, 32 * WARPS, smem, stream>>>(keys, d, rows, groups, bits, nullptr, nullptr, order, offsets);
            FMB_LAUNCH_CHECK();
            return FMB_OK;
        }
    }
    FMB_CUDA_CHECK(opt_in_shared_memory((const void*)k_group_place<K, false, DIGIT, WARPS>, most));
    int32_t* const totals = scratch + (long long)ctas * width;
    FMB_CUDA_CHECK(launch(k_group_count<K, DIGIT, WARPS>, ctas, 32 * WARPS, 0, keys, d, rows, groups, scratch));
    FMB_LAUNCH_CHECK();
    FMB_CUDA_CHECK(launch(k_group_scan<DIGIT>, ceil_div(width, 32), 1024, 0, scratch, totals, ctas, width));
    FMB_LAUNCH_CHECK();
    FMB_CUDA_CHECK(launch(k_group_place<K, false, DIGIT, WARPS>, ctas, 32 * WARPS, smem, keys, d, rows, groups, bits, scratch, totals, order, offsets));
    FMB_LAUNCH_CHECK();
    return FMB_OK;
}

// Tokens by value: one pass where the table holds every value, else one over the lower half of their bits and one over the upper half,
// which keeps the order that the first has made.
int lower_bits(int vocabulary) { return vocabulary <= FMB_MAX_GROUPS ? 0 : (33 - __builtin_clz(vocabulary)) / 2; }
// CTAs of eight warps, while that spreads the rows over more SMs
int warps_of(long long rows) { return rows <= 148ll * 8 * kFewWarps * kRowsPerWarp ? kFewWarps : kWarps; }
long long table_size(long long rows, int width) {
    const long long per_cta = warps_of(rows) * kRowsPerWarp;
    return ((rows + per_cta - 1) / per_cta + 1) * width;
}

template <typename K>
int sort_digit(const K* keys, const Digit& d, long long rows, int groups, int32_t* order, int32_t* scratch, cudaStream_t stream) {
    return warps_of(rows) == kWarps ? sort_pass<K, true, kWarps>(keys, d, rows, groups, order, nullptr, scratch, stream)
                                    : sort_pass<K, true, kFewWarps>(keys, d, rows, groups, order, nullptr, scratch, stream);
}

// Few rows: the place of each is the number of those before it, for which eight lanes count a row's share of all, four at a time. One launch
// for any vocabulary, each CTA with 32 rows (1,928 rows by two passes of one CTA: 8 us more; by one CTA alone 75 us more).
constexpr int kFewRows = kRowsPerCta, kRankRows = 32;

template <typename K>
__global__ void __launch_bounds__(8 * kRankRows)
k_rank_tokens(const K* tokens, int rows, int vocabulary, int32_t* __restrict__ order, int32_t* __restrict__ keys) {
    __shared__ int4 all[kFewRows / 4];
    let_next_come();
    kernels_before(tokens);
    int* const key = reinterpret_cast<int*>(all);
    const int quads = (rows + 3) / 4;
#pragma unroll 4
    for (int i = threadIdx.x; i < 4 * quads; i += 8 * kRankRows) key[i] = i < rows ? group_of(tokens[i], vocabulary) : 0x7fffffff;
    __syncthreads();
    const int i = blockIdx.x * kRankRows + (threadIdx.x >> 3), mine = i < rows ? key[i] : 0, own = i / 4;
    int before = 0;
    // a key as large as this one counts where its row comes before
#pragma unroll 4
    for (int q = threadIdx.x & 7; q < quads; q += 8) {
        const int4 k = all[q];
        const int bound = mine + (q < own);
        before += (k.x < bound) + (k.y < bound) + (k.z < bound) + (k.w < bound);
        if (q == own) before += (i % 4 > 0 && k.x == mine) + (i % 4 > 1 && k.y == mine) + (i % 4 > 2 && k.z == mine);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
    if (i < rows && (threadIdx.x & 7) == 0) {
        order[before] = i;
        keys[before] = mine;
    }
}

template <typename K>
int sort_tokens(const K* tokens, long long rows, int vocabulary, int32_t* order, int32_t* keys, int32_t* scratch, cudaStream_t stream) {
    if (rows <= kFewRows) {
        FMB_CUDA_CHECK(launch_early(k_rank_tokens<K>, ceil_div(rows, kRankRows), 8 * kRankRows, 0, stream, tokens, (int)rows, vocabulary, order, keys));
        FMB_LAUNCH_CHECK();
        return FMB_OK;
    }
    const int low = lower_bits(vocabulary);
    if (low == 0) return sort_digit(tokens, Digit{nullptr, keys, vocabulary, 0, -1}, rows, vocabulary, order, scratch, stream);
    int32_t* const table = scratch + rows;
    const int rc = sort_digit(tokens, Digit{nullptr, nullptr, vocabulary, 0, (1 << low) - 1}, rows, (1 << low) - 1, scratch, table, stream);
    return rc ? rc : sort_digit(tokens, Digit{scratch, keys, vocabulary, low, -1}, rows, vocabulary >> low, order, table, stream);
}

}  // namespace

}  // namespace fmb

using namespace fmb;

extern "C" FMB_API long long fmb_group_rows_scratch(long long rows, int groups) {
    if (rows <= kRowsPerCta || groups < 1) return 0;
    return ((rows + kRowsPerCta - 1) / kRowsPerCta + 1) * (groups + 1);
}

extern "C" FMB_API int fmb_group_rows(const void* keys, int key_bytes, long long rows, int groups, int32_t* order,
                                      int32_t* offsets, int32_t* scratch, fmb_stream_t stream) {
    FMB_REQUIRE(groups >= 1 && groups <= FMB_MAX_GROUPS, "fmb_group_rows: 1 to FMB_MAX_GROUPS groups");
    FMB_REQUIRE(rows >= 0 && rows < (1ll << 31) - kRowsPerCta, "fmb_group_rows: too many rows");
    FMB_REQUIRE(offsets && (rows == 0 || (keys && order)), "fmb_group_rows: null argument");
    FMB_REQUIRE(scratch || fmb_group_rows_scratch(rows, groups) == 0, "fmb_group_rows: null scratch");
    FMB_REQUIRE(key_bytes == 4 || key_bytes == 8, "fmb_group_rows: keys of 4 or 8 bytes");
    if (key_bytes == 4)
        return sort_pass<int32_t, false, kWarps>((const int32_t*)keys, Digit{}, rows, groups, order, offsets, scratch, (cudaStream_t)stream);
    return sort_pass<long long, false, kWarps>((const long long*)keys, Digit{}, rows, groups, order, offsets, scratch, (cudaStream_t)stream);
}

extern "C" FMB_API long long fmb_sort_tokens_scratch(long long rows, int vocabulary) {
    if (rows <= kFewRows || vocabulary < 1 || vocabulary > FMB_MAX_VOCABULARY) return 0;
    const int low = lower_bits(vocabulary);
    if (low == 0) return table_size(rows, vocabulary + 1);
    return rows + table_size(rows, std::max(1 << low, (vocabulary >> low) + 1));
}

extern "C" FMB_API int fmb_sort_tokens(const void* tokens, int token_bytes, long long rows, int vocabulary, int32_t* order,
                                       int32_t* keys, int32_t* scratch, fmb_stream_t stream) {
    FMB_REQUIRE(vocabulary >= 1 && vocabulary <= FMB_MAX_VOCABULARY, "fmb_sort_tokens: 1 to FMB_MAX_VOCABULARY tokens");
    FMB_REQUIRE(rows >= 0 && rows < (1ll << 31) - kRowsPerCta, "fmb_sort_tokens: too many rows");
    FMB_REQUIRE(token_bytes == 4 || token_bytes == 8, "fmb_sort_tokens: tokens of 4 or 8 bytes");
    if (rows == 0) return FMB_OK;
    FMB_REQUIRE(tokens && order && keys, "fmb_sort_tokens: null argument");
    FMB_REQUIRE(scratch || fmb_sort_tokens_scratch(rows, vocabulary) == 0, "fmb_sort_tokens: null scratch");
    if (token_bytes == 4) return sort_tokens((const int32_t*)tokens, rows, vocabulary, order, keys, scratch, (cudaStream_t)stream);
    return sort_tokens((const long long*)tokens, rows, vocabulary, order, keys, scratch, (cudaStream_t)stream);
}
