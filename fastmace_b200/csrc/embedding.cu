// Rows of a table by token, and the table's gradient.
//
//   lookup:    out[r] = scale E[t(r)]
//   gradient:  dE[v] = scale sum of dy[r] over the rows r of token v, from rows sorted by token (fmb_sort_tokens)
//
// The gradient is a sum over runs of equal tokens. The sorted places are cut into chunks of one size, whatever the runs are, and a
// warp sums a chunk's rows for a slab of columns: a word in thousands of places costs as much per row as one in two. A run that lies
// within a chunk is written at once; the parts of one that does not go to scratch, and a second kernel adds them in their order.
// Other warps of the first launch write the zeros of tokens without rows. No atomics: the same call gives the same bits.
//
// Bound by memory: every row is read once and every row of the table written once.

#include "early.cuh"
#include "eight.cuh"

#include <algorithm>
#include <type_traits>

namespace fmb {
namespace emb {

namespace {

using eight::rounded;
using eight::to_float;

// N values side by side in one load or store of up to 16 bytes
template <typename T, int N> struct alignas(N * sizeof(T)) Pack { T v[N]; };

// (what is written is not read again soon: 200,000 rows of 512 fp16 values 71 us, and 61 so)
template <typename T, int N>
__device__ __forceinline__ void store_streaming(T* to, const Pack<T, N>& v) {
    if constexpr (N * sizeof(T) == 16) __stcs(reinterpret_cast<uint4*>(to), *reinterpret_cast<const uint4*>(&v));
    else if constexpr (N * sizeof(T) == 8) __stcs(reinterpret_cast<uint2*>(to), *reinterpret_cast<const uint2*>(&v));
    else *reinterpret_cast<Pack<T, N>*>(to) = v;
}

// -------------------------------------------------------------------------------------------------------------- lookup

// Lanes that share a row: as many as it has packs of N values, a power of two up to 32; a warp has ROWS times 32 / lanes rows at a time, and a
// lane four packs on their way. WIDE: rows start at multiples of a pack; else a pack is eight values by the words that they lie in.
template <typename T, typename O, typename K, int N, int ROWS, bool WIDE>
__global__ void __launch_bounds__(256)
k_embedding(fmb_embedding_t a, int lanes) {
    constexpr int kOfRow = 4 / ROWS;             // packs of a row on their way
    static_assert(WIDE || N == eight::kEach, "eight values by words");
    using In = typename std::conditional<WIDE, Pack<T, N>, eight::Raw<T>>::type;
    const int lane = threadIdx.x & 31, part = lane & (lanes - 1), per_warp = 32 / lanes;
    const long long warp = (blockIdx.x * 256ll + threadIdx.x) >> 5, warps = gridDim.x * 8ll;
    const float scale = (float)a.scale;
    const int packs = a.width / N;
    for (long long r0 = warp * per_warp * ROWS + lane / lanes; r0 < a.rows; r0 += warps * per_warp * ROWS) {
        K token[ROWS];
        bool live[ROWS];
#pragma unroll
        for (int q = 0; q < ROWS; ++q) token[q] = r0 + q * per_warp < a.rows ? ((const K*)a.tokens)[r0 + q * per_warp] : (K)-1;
#pragma unroll
        for (int q = 0; q < ROWS; ++q) live[q] = token[q] >= 0 && token[q] < (K)a.vocabulary;
        auto from = [&](int q) { return (const T*)a.source + (live[q] ? (long long)token[q] : 0) * a.source_stride; };
        auto to = [&](int q) { return (O*)a.out + (r0 + q * per_warp) * a.out_stride; };
        auto written = [&](int q) { return r0 + q * per_warp < a.rows && (live[q] || a.zero_rest); };
        for (int c = part; c < packs; c += kOfRow * lanes) {
            In in[ROWS][kOfRow];
#pragma unroll
            for (int q = 0; q < ROWS; ++q)
#pragma unroll
                for (int j = 0; j < kOfRow; ++j) {
                    if (live[q] && c + j * lanes < packs) {
                        if constexpr (WIDE) in[q][j] = *reinterpret_cast<const In*>(from(q) + (c + j * lanes) * N);
                        else in[q][j] = eight::load<T, false>(from(q) + (c + j * lanes) * N, N);
                    }
                }
#pragma unroll
            for (int q = 0; q < ROWS; ++q) {
                if (!written(q)) continue;
#pragma unroll
                for (int j = 0; j < kOfRow; ++j) {
                    if (c + j * lanes >= packs) break;
                    O* const at = to(q) + (c + j * lanes) * N;
                    if constexpr (WIDE) {
                        Pack<O, N> out;
#pragma unroll
                        for (int i = 0; i < N; ++i) out.v[i] = rounded<O>(live[q] ? scale * to_float(in[q][j].v[i]) : 0.0f);
                        store_streaming<O, N>(at, out);
                    } else {
                        float x[N] = {};
                        if (live[q]) eight::unpack<T>(in[q][j], x);
#pragma unroll
                        for (int i = 0; i < N; ++i) x[i] = live[q] ? scale * x[i] : 0.0f;
                        eight::store<O, false>(at, N, x);
                    }
                }
            }
        }
        // the columns behind the last whole pack
        for (int c = packs * N + part; c < a.width; c += lanes)
#pragma unroll
            for (int q = 0; q < ROWS; ++q)
                if (written(q)) to(q)[c] = rounded<O>(live[q] ? scale * to_float(from(q)[c]) : 0.0f);
    }
}

bool starts_at(const void* base, long long stride, int bytes, int values) {
    return ((uintptr_t)base & (uintptr_t)(bytes * values - 1)) == 0 && stride % values == 0;
}

template <typename T, typename O, typename K, int N, bool WIDE>
int lookup_by(const fmb_embedding_t& a, cudaStream_t stream) {
    const int packs = std::max(1, a.width / N);
    int lanes = 1;
    while (lanes < 32 && lanes < packs) lanes *= 2;
    // rows at a time: as many as give a lane four packs, where that leaves work for every SM (300,000 rows of 128 values: 82 us with one, 27 with four)
    const int of_lane = ceil_div(packs, lanes), rows = of_lane > 2 || (long long)a.rows * lanes < 148 * 2048 ? 1 : of_lane > 1 ? 2 : 4;
    const int grid = std::min(ceil_div((long long)ceil_div(a.rows, rows) * lanes, 256), 1 << 20);
    const auto kernel = rows == 1 ? k_embedding<T, O, K, N, 1, WIDE> : rows == 2 ? k_embedding<T, O, K, N, 2, WIDE> : k_embedding<T, O, K, N, 4, WIDE>;
    kernel<<<grid, 256, 0, stream>>>(a, lanes);
    FMB_LAUNCH_CHECK();
    return FMB_OK;
}

// packs of 16 bytes of the larger type where rows start at multiples of them, of four values where they start at those
template <typename T, typename O, typename K>
int lookup(const fmb_embedding_t& a, cudaStream_t stream) {
    constexpr int kPack = sizeof(T) == 4 || sizeof(O) == 4 ? 4 : 8;
    auto by = [&](int n) { return starts_at(a.source, a.source_stride, sizeof(T), n) && starts_at(a.out, a.out_stride, sizeof(O), n); };
    return by(kPack) ? lookup_by<T, O, K, kPack, true>(a, stream) : by(4) ? lookup_by<T, O, K, 4, true>(a, stream) : lookup_by<T, O, K, 8, false>(a, stream);
}

template <typename T, typename O>
int lookup(const fmb_embedding_t& a, cudaStream_t stream) {
    return a.token_bytes == 4 ? lookup<T, O, int32_t>(a, stream) : lookup<T, O, long long>(a, stream);
}

template <typename T>
int lookup(const fmb_embedding_t& a, cudaStream_t stream) {
    return a.out_type == FMB_TYPE_F32    ? lookup<T, float>(a, stream)
           : a.out_type == FMB_TYPE_BF16 ? lookup<T, __nv_bfloat16>(a, stream)
                                         : lookup<T, __half>(a, stream);
}

// ------------------------------------------------------------------------------------------------------------ gradient

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kUnroll = 8;                       // rows on their way

// Columns of a slab: of every lane N side by side (VEC), or N that are 32 apart, where rows do not start at multiples of a pack
template <bool VEC, int N>
__device__ __forceinline__ int column(int slab, int i) {
    const int lane = threadIdx.x & 31;
    return slab * 32 * N + (VEC ? lane * N + i : lane + 32 * i);
}

// A lane's N values of a row as they are in memory, 16 bytes (fp32, four) or up to 16, so that a row waits in few registers
template <typename T, bool VEC, int N>
__device__ __forceinline__ uint4 load_columns(const T* __restrict__ row, int slab, int width) {
    const int c0 = column<VEC, N>(slab, 0);
    if (VEC && c0 + N <= width) return __ldg(reinterpret_cast<const uint4*>(row + c0));
    uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = column<VEC, N>(slab, i);
        if constexpr (sizeof(T) == 4) v[i] = c < width ? __ldg(reinterpret_cast<const uint32_t*>(row) + c) : 0u;
        else v[i / 2] |= (c < width ? (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(row) + c) : 0u) << (16 * (i % 2));
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
}

template <typename T> __device__ __forceinline__ float2 two_of(uint32_t v);
template <> __device__ __forceinline__ float2 two_of<__nv_bfloat16>(uint32_t v) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)); }
template <> __device__ __forceinline__ float2 two_of<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }

// a lane's N values
template <typename T, int N>
__device__ __forceinline__ void unpack_columns(float (&out)[N], const uint4& x) {
    if constexpr (sizeof(T) == 4) {
        out[0] = __uint_as_float(x.x);
        out[1] = __uint_as_float(x.y);
        out[2] = __uint_as_float(x.z);
        out[3] = __uint_as_float(x.w);
    } else {
        const uint32_t v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 two = two_of<T>(v[i / 2]);
            out[i] = two.x;
            out[i + 1] = two.y;
        }
    }
}

template <typename T, int N>
__device__ __forceinline__ void add_columns(float (&sum)[N], const uint4& x) {
    float v[N];
    unpack_columns<T, N>(v, x);
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i] += v[i];
}

struct Sums {
    fmb_embedding_t a;
    int chunk, chunks, slabs;                    // rows of a CTA's chunk, kWarps shares of them
    int wide_out;                                // rows of the table start at multiples of 16 bytes
    long long part_stride;                       // floats of a part in scratch: the width, filled up to a multiple of four
    unsigned zero_ctas, zero_shares;             // CTAs that write zeros, before those that sum, and of how many they share a row's columns
};

// first place from `low` on whose key is not less than v, by a warp: 32 places of what is left at a time
__device__ __forceinline__ int lower_bound(const int32_t* __restrict__ keys, int low, int high, int v) {
    const int lane = threadIdx.x & 31;
    while (low < high) {
        const int step = (high - low + 31) / 32, at = min(low + lane * step, high - 1);
        // of falling runs of "less", the last probe that is
        const int less = __popc(__ballot_sync(0xffffffffu, low + lane * step < high && __ldg(keys + at) < v));
        if (less == 0) return low;
        const int last = low + (less - 1) * step;
        high = min(high, last + step);
        low = last + 1;
    }
    return low;
}

// Zeros for the tokens without rows: kZeroTokens of them and a share of the columns by a CTA. Warp 0 finds out which have rows.
constexpr int kZeroTokens = 32;

__device__ __forceinline__ void write_zeros(const Sums& p) {
    __shared__ uint32_t present;
    const fmb_embedding_t& a = p.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int32_t* const keys = (const int32_t*)a.tokens;
    const int first = (int)(blockIdx.x / p.zero_shares) * kZeroTokens, last = min(first + kZeroTokens, a.vocabulary);
    if (warp == 0) {
        const int from = lower_bound(keys, 0, a.rows, first), to = lower_bound(keys, from, a.rows, last);
        uint32_t seen = 0;
        if (to - from > 256) {
            // tokens of many rows: a lane looks for its own
            int low = from, high = first + lane < last ? to : from;
            while (low < high) {
                const int mid = (int)(((unsigned)low + (unsigned)high) >> 1);
                if (__ldg(keys + mid) < first + lane) low = mid + 1; else high = mid;
            }
            seen = __ballot_sync(0xffffffffu, first + lane < last && low < to && __ldg(keys + low) == first + lane);
        } else {
            for (int at = from + lane; at < to; at += 32) seen |= 1u << ((__ldg(keys + at) - first) & 31);
            seen = __reduce_or_sync(0xffffffffu, seen);
        }
        if (lane == 0) present = seen;
    }
    __syncthreads();
    const int share = blockIdx.x % p.zero_shares, units = p.wide_out ? a.width / 4 : a.width;
    const int begin = (int)((long long)units * share / p.zero_shares), end = (int)((long long)units * (share + 1) / p.zero_shares);
    for (int v = first + warp; v < last; v += kWarps) {
        if (present >> (v - first) & 1) continue;
        float* const out = (float*)a.out + v * a.out_stride;
        if (p.wide_out) {
            for (int c = begin + lane; c < end; c += 32) reinterpret_cast<float4*>(out)[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (share == p.zero_shares - 1 && lane < a.width % 4) out[4 * units + lane] = 0.0f;
        } else {
            for (int c = begin + lane; c < end; c += 32) out[c] = 0.0f;
        }
    }
}

// out (+)= scale sum, or a part as it is
template <bool VEC, int N>
__device__ __forceinline__ void write_sums(const Sums& p, int slab, float* out, bool part, const float (&sum)[N]) {
    const fmb_embedding_t& a = p.a;
    const float scale = (float)a.scale;
    const bool wide = VEC && (part || p.wide_out);
#pragma unroll
    for (int i0 = 0; i0 < N; i0 += 4) {
        const int c0 = column<VEC, N>(slab, i0);
        if (wide && c0 + 4 <= a.width) {
            float4* const to = reinterpret_cast<float4*>(out + c0);
            float4 s = make_float4(sum[i0], sum[i0 + 1], sum[i0 + 2], sum[i0 + 3]);
            if (!part) {
                const float4 old = a.accumulate ? *to : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                s = make_float4(old.x + scale * s.x, old.y + scale * s.y, old.z + scale * s.z, old.w + scale * s.w);
            }
            *to = s;
        } else {
#pragma unroll
            for (int i = i0; i < i0 + 4; ++i) {
                const int c = column<VEC, N>(slab, i);
                if (c < a.width) out[c] = part ? sum[i] : (a.accumulate ? out[c] : 0.0f) + scale * sum[i];
            }
        }
    }
}

// A chunk's places are shared by the CTA's warps in kWarps runs of their own. The parts of a run of equal keys that goes over a warp's
// end meet in shared memory; the parts of one that goes over the chunk's end go to scratch, the first of a chunk's two places
// holding what a run has that began before it, the other what one has that begins in it and goes on.
template <typename T, bool VEC, int N>
__global__ void __launch_bounds__(kThreads, 3)
k_embedding_sums(Sums p) {
    let_next_come();
    kernels_before(p.a.tokens, p.a.order, p.a.source);
    if (blockIdx.x < p.zero_ctas) {              // the first, since their searches take long and their writes little
        write_zeros(p);
        return;
    }
    __shared__ float parts[2][kWarps][N][32];    // of each warp: of the run that it begins with, of the one that it ends with
    __shared__ int states[kWarps][2];
    const fmb_embedding_t& a = p.a;
    const int32_t* const keys = (const int32_t*)a.tokens;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned unit = blockIdx.x - p.zero_ctas;
    const int chunk = (int)(unit / p.slabs), slab = (int)(unit % p.slabs);
    const int chunk_begin = chunk * p.chunk, chunk_end = min(a.rows, chunk_begin + p.chunk), share = p.chunk / kWarps;
    const int begin = min(chunk_end, chunk_begin + warp * share), end = min(chunk_end, begin + share);
    // of a run: its key, and whether it began before this warp's rows
    int key = begin < end ? __ldg(keys + begin) : a.vocabulary;
    bool before = begin > 0 && begin < end && __ldg(keys + begin - 1) == key;
    const bool has_first = before;
    bool first_ends = false;                     // the run that began before ends here
    float sum[N];
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i] = 0.0f;
    auto keep = [&](int which) {
#pragma unroll
        for (int i = 0; i < N; ++i) parts[which][warp][i][lane] = sum[i];
    };
    auto flush = [&]() {
        if (before) {
            keep(0);
            first_ends = true;
        } else if (key >= 0 && key < a.vocabulary) {
            write_sums<VEC, N>(p, slab, (float*)a.out + key * a.out_stride, false, sum);
        }
    };

    for (int p0 = begin; p0 < end; p0 += 32) {
        const int mine = p0 + lane < end ? __ldg(keys + p0 + lane) : a.vocabulary, count = min(32, end - p0);
        int row = p0 + lane < end ? __ldg(a.order + p0 + lane) : -1;
        if (row >= a.rows || mine < 0 || mine >= a.vocabulary) row = -1;
        for (int j0 = 0; j0 < count; j0 += kUnroll) {
            uint4 x[kUnroll];
#pragma unroll
            for (int j = 0; j < kUnroll; ++j) {
                const int r = __shfl_sync(0xffffffffu, row, j0 + j);
                x[j] = r >= 0 ? load_columns<T, VEC, N>((const T*)a.source + r * a.source_stride, slab, a.width) : make_uint4(0, 0, 0, 0);
            }
            // Eight rows of the run that is being added up: as a tree, so that a long run's sum goes through an eighth of the additions (884,736 rows of
            // 128 fp32 by 89 tokens, one after the other: 3.0e-7 of the norm off in 83 us; so 1.4e-7 in 80)
            if (j0 + kUnroll <= count && __shfl_sync(0xffffffffu, mine, j0 + kUnroll - 1) == key) {
                float tree[kUnroll / 2][N];
#pragma unroll
                for (int j = 0; j < kUnroll; j += 2) {
                    unpack_columns<T, N>(tree[j / 2], x[j]);
                    add_columns<T, N>(tree[j / 2], x[j + 1]);
                    if (j % 4 == 2) {
#pragma unroll
                        for (int i = 0; i < N; ++i) tree[j / 2 - 1][i] += tree[j / 2][i];
                    }
                }
#pragma unroll
                for (int i = 0; i < N; ++i) sum[i] += tree[0][i] + tree[2][i];
                continue;
            }
#pragma unroll
            for (int j = 0; j < kUnroll; ++j) {
                const int next = __shfl_sync(0xffffffffu, mine, j0 + j);
                if (j0 + j < count && next != key) {
                    flush();
                    key = next;
                    before = false;
#pragma unroll
                    for (int i = 0; i < N; ++i) sum[i] = 0.0f;
                }
                add_columns<T, N>(sum, x[j]);
            }
        }
    }
    const bool after = begin < end && end < a.rows && __ldg(keys + end) == key;
    bool has_last = false;
    if (begin < end) {
        if (before) {
            keep(0);
            first_ends = !after;
        } else if (after) {
            keep(1);
            has_last = true;
        } else {
            flush();
        }
    }
    // bits: a run that began before, which ends here; one that goes on
    if (lane == 0) {
        states[warp][0] = (has_first ? 1 : 0) | (first_ends ? 2 : 0) | (has_last ? 4 : 0);
        states[warp][1] = key;
    }
    __syncthreads();
    // The warps' parts in their order. Each warp adds up the runs that end in the warps of its turn: the run that a warp ends with is
    // followed through the ones behind it, by that warp; the run that the chunk begins with by warp 0.
    auto follow = [&](int w0) {
        // (sum holds what the run has so far)
        bool ended = false;
        int w = w0;
        for (; w < kWarps && !ended && (states[w][0] & 1); ++w) {
#pragma unroll
            for (int i = 0; i < N; ++i) sum[i] += parts[0][w][i][lane];
            ended = states[w][0] & 2;
        }
        return ended;
    };
    if (warp == 0 && (states[0][0] & 1)) {
        const int run = __ldg(keys + chunk_begin);
#pragma unroll
        for (int i = 0; i < N; ++i) sum[i] = 0.0f;
        follow(0);
        if (run >= 0 && run < a.vocabulary) write_sums<VEC, N>(p, slab, a.scratch + 2ll * chunk * p.part_stride, true, sum);
    }
    if (states[warp][0] & 4) {
        const int run = states[warp][1];
#pragma unroll
        for (int i = 0; i < N; ++i) sum[i] = parts[1][warp][i][lane];
        const bool ended = follow(warp + 1);
        if (run >= 0 && run < a.vocabulary) {
            if (ended) write_sums<VEC, N>(p, slab, (float*)a.out + run * a.out_stride, false, sum);
            else write_sums<VEC, N>(p, slab, a.scratch + (2ll * chunk + 1) * p.part_stride, true, sum);
        }
    }
}

// The runs that go over the end of the chunk in which they begin: their parts, added in the order of the chunks. A CTA has every
// gridDim.x-th chunk; a run's parts are shared by warps, and slabs of 128 columns by others.
constexpr int kJoinWarps = 32, kJoinList = 64;

__global__ void __launch_bounds__(kJoinWarps * 32)
k_embedding_join(Sums p) {
    constexpr int kThreads = 32 * kJoinWarps;
    __shared__ int list[kJoinList], count;
    __shared__ float4 sums[kJoinWarps][32];
    kernels_before(p.a.tokens, p.a.scratch);
    const fmb_embedding_t& a = p.a;
    const int32_t* const keys = (const int32_t*)a.tokens;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float scale = (float)a.scale;
    const int slabs = (a.width + 127) / 128;
    // warps of a slab: as many as leave none without work in a pass over the slabs
    int shares = 1;
    while (shares < kJoinWarps && 2 * shares * slabs <= kJoinWarps) shares *= 2;
    for (int c0 = blockIdx.x; c0 < p.chunks; c0 += gridDim.x * kJoinList) {
        __syncthreads();
        if (threadIdx.x == 0) count = 0;
        __syncthreads();
        if (threadIdx.x < kJoinList) {
            const long long chunk = c0 + (long long)threadIdx.x * gridDim.x;
            if (chunk < p.chunks - 1) {                           // the last one ends with the rows
                const int begin = (int)chunk * p.chunk, end = begin + p.chunk, key = __ldg(keys + end - 1);
                const bool begins = begin == 0 || __ldg(keys + begin - 1) != key || __ldg(keys + begin) != key;
                if (key >= 0 && key < a.vocabulary && __ldg(keys + end) == key && begins) list[atomicAdd(&count, 1)] = (int)chunk;
            }
        }
        __syncthreads();
        for (int q = 0; q < count; ++q) {
            const int chunk = list[q], key = __ldg(keys + (chunk + 1) * p.chunk - 1);
            // the chunks behind it that begin with the run, 1,024 looked at together
            int parts = 1;
            for (int first = chunk + 1, some = kThreads; some == kThreads; first += kThreads) {
                some = __syncthreads_count(first + (int)threadIdx.x < p.chunks && __ldg(keys + (long long)(first + threadIdx.x) * p.chunk) == key);
                parts += some;
            }
            for (int s0 = 0; s0 < slabs; s0 += kJoinWarps / shares) {
                const int slab = s0 + warp / shares, part = warp % shares, c = slab * 128 + 4 * lane;
                float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (c < a.width) {
                    const int from = (int)((long long)parts * part / shares), to = (int)((long long)parts * (part + 1) / shares);
                    for (int u0 = from; u0 < to; u0 += 8) {
                        float4 x[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            // the first part is what its chunk ends with, the others what theirs begin with
                            const int u = u0 + j;
                            if (u < to) x[j] = *reinterpret_cast<const float4*>(a.scratch + (2ll * (chunk + u) + (u == 0)) * p.part_stride + c);
                        }
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            if (u0 + j >= to) break;
                            sum.x += x[j].x; sum.y += x[j].y; sum.z += x[j].z; sum.w += x[j].w;
                        }
                    }
                }
                __syncthreads();
                sums[warp][lane] = sum;
                __syncthreads();
                if (part > 0 || c >= a.width) continue;
                for (int w = 1; w < shares; ++w) {
                    const float4 x = sums[warp + w][lane];
                    sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
                }
                float* const out = (float*)a.out + key * a.out_stride + c;
                const float v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (c + i < a.width) out[i] = (a.accumulate ? out[i] : 0.0f) + scale * v[i];
            }
        }
    }
}

// Rows per chunk: kWarps shares that make enough warps for 24 on every SM, and as few parts as that leaves; a share has between 8 rows,
// what a warp has on their way, and 256. By sizes and type alone, with the slabs of rows at multiples of 16 bytes: the order of the sums and the
// room for their parts do not depend on where the rows lie.
int chunk_rows(const fmb_embedding_t& a) {
    const long long rows = (long long)a.rows * ceil_div(a.width, a.type == FMB_TYPE_F32 ? 128 : 256) / (148 * 24) + 1;
    return kWarps * (int)std::min(256ll, std::max(8ll, (rows + 7) / 8 * 8));
}

bool packed(const fmb_embedding_t& a) {
    return starts_at(a.source, a.source_stride, a.type == FMB_TYPE_F32 ? 4 : 2, a.type == FMB_TYPE_F32 ? 4 : 8);
}

template <typename T>
int gradient(const fmb_embedding_t& a, cudaStream_t stream) {
    constexpr int kPack = 16 / sizeof(T);
    Sums p;
    p.a = a;
    p.slabs = ceil_div(a.width, a.type != FMB_TYPE_F32 && packed(a) ? 256 : 128);
    p.chunk = chunk_rows(a);
    p.chunks = ceil_div(a.rows, p.chunk);
    p.wide_out = starts_at(a.out, a.out_stride, 4, 4);
    p.part_stride = (a.width + 3) / 4 * 4;
    // two CTAs for every SM, as far as a share keeps 512 columns
    const int zero_groups = ceil_div(a.vocabulary, kZeroTokens);
    p.zero_shares = std::max(1, std::min(ceil_div(2 * 148, zero_groups), a.width / 512));
    p.zero_ctas = a.accumulate ? 0 : zero_groups * p.zero_shares;
    const long long ctas = p.zero_ctas + (long long)p.chunks * p.slabs;
    FMB_REQUIRE(ctas < (1ll << 31), "fmb_embedding_gradient: too many sums");
    if (ctas > 0) {
        FMB_CUDA_CHECK(launch_early(packed(a) ? k_embedding_sums<T, true, kPack> : k_embedding_sums<T, false, 4>, (unsigned)ctas, kThreads, 0, stream, p));
        FMB_LAUNCH_CHECK();
    }
    if (p.chunks > 1) {
        FMB_CUDA_CHECK(launch_early(k_embedding_join, std::min(p.chunks, 148), kJoinWarps * 32, 0, stream, p));
        FMB_LAUNCH_CHECK();
    }
    return FMB_OK;
}

int check(const fmb_embedding_t* a) {
    FMB_REQUIRE(a, "embedding: null argument");
    FMB_REQUIRE(a->type >= FMB_TYPE_F32 && a->type <= FMB_TYPE_F16, "embedding: type");
    FMB_REQUIRE(a->vocabulary >= 1 && a->vocabulary <= FMB_MAX_VOCABULARY, "embedding: 1 to FMB_MAX_VOCABULARY tokens");
    FMB_REQUIRE(a->rows >= 0 && a->rows <= (1 << 30), "embedding: more than 2^30 rows");
    FMB_REQUIRE(a->width >= 1 && a->width <= (1 << 20), "embedding: 1 to 2^20 columns");
    FMB_REQUIRE(a->rows == 0 || (a->tokens && a->source), "embedding: null argument");
    return FMB_OK;
}

}  // namespace

}  // namespace emb
}  // namespace fmb

using namespace fmb;
using namespace fmb::emb;

extern "C" FMB_API int fmb_embedding(const fmb_embedding_t* a, fmb_stream_t stream) {
    const int rc = check(a);
    if (rc) return rc;
    FMB_REQUIRE(a->out_type >= FMB_TYPE_F32 && a->out_type <= FMB_TYPE_F16, "fmb_embedding: type of the rows");
    FMB_REQUIRE(a->token_bytes == 4 || a->token_bytes == 8, "fmb_embedding: tokens of 4 or 8 bytes");
    if (a->rows == 0) return FMB_OK;
    FMB_REQUIRE(a->out, "fmb_embedding: null argument");
    FMB_REQUIRE((a->vocabulary == 1 || a->source_stride >= a->width) && (a->rows == 1 || a->out_stride >= a->width), "fmb_embedding: rows overlap");
    return a->type == FMB_TYPE_F32    ? lookup<float>(*a, (cudaStream_t)stream)
           : a->type == FMB_TYPE_BF16 ? lookup<__nv_bfloat16>(*a, (cudaStream_t)stream)
                                      : lookup<__half>(*a, (cudaStream_t)stream);
}

extern "C" FMB_API long long fmb_embedding_gradient_scratch(const fmb_embedding_t* a) {
    if (!a || a->rows < 1 || a->width < 1 || a->type < FMB_TYPE_F32 || a->type > FMB_TYPE_F16) return 0;
    const int chunk = chunk_rows(*a);
    return a->rows <= chunk ? 0 : 2ll * ceil_div(a->rows, chunk) * ((a->width + 3) / 4 * 4);
}

extern "C" FMB_API int fmb_embedding_gradient(const fmb_embedding_t* a, fmb_stream_t stream) {
    const int rc = check(a);
    if (rc) return rc;
    FMB_REQUIRE(a->out && (a->rows == 0 || a->order), "fmb_embedding_gradient: null argument");
    FMB_REQUIRE((a->rows <= 1 || a->source_stride >= a->width) && (a->vocabulary == 1 || a->out_stride >= a->width), "fmb_embedding_gradient: rows overlap");
    FMB_REQUIRE(a->scratch || fmb_embedding_gradient_scratch(a) == 0, "fmb_embedding_gradient: null scratch");
    FMB_REQUIRE(((uintptr_t)a->scratch & 15) == 0, "fmb_embedding_gradient: scratch starts at a multiple of 16 bytes");
    return a->type == FMB_TYPE_F32    ? gradient<float>(*a, (cudaStream_t)stream)
           : a->type == FMB_TYPE_BF16 ? gradient<__nv_bfloat16>(*a, (cudaStream_t)stream)
                                      : gradient<__half>(*a, (cudaStream_t)stream);
}
