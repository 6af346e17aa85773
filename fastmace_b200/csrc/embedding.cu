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

#include "grouped.cuh"

#include <algorithm>

namespace fmb {
namespace emb {

namespace {

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T rounded(float x) { return grp::from_float<T>(x); }
template <> __device__ __forceinline__ float rounded<float>(float x) { return x; }

// N values side by side in one load or store of up to 16 bytes
template <typename T, int N> struct alignas(N * sizeof(T)) Pack { T v[N]; };

// -------------------------------------------------------------------------------------------------------------- lookup

// Lanes that share a row: as many as it has packs, a power of two up to 32; a warp has 32 / lanes rows at a time and four packs a lane
// on their way. N = 1 where rows do not start at multiples of a pack.
template <typename T, typename O, typename K, int N>
__global__ void __launch_bounds__(256)
k_embedding(fmb_embedding_t a, int lanes) {
    const int lane = threadIdx.x & 31, part = lane & (lanes - 1), per_warp = 32 / lanes;
    const long long warp = (blockIdx.x * 256ll + threadIdx.x) >> 5, warps = gridDim.x * 8ll;
    const float scale = (float)a.scale;
    const int packs = a.width / N;
    for (long long r = warp * per_warp + lane / lanes; r < a.rows; r += warps * per_warp) {
        const K token = ((const K*)a.tokens)[r];
        const bool live = token >= 0 && token < (K)a.vocabulary;
        if (!live && !a.zero_rest) continue;
        const T* const from = (const T*)a.source + (live ? (long long)token : 0) * a.source_stride;
        O* const to = (O*)a.out + r * a.out_stride;
        for (int c = part; c < packs; c += 4 * lanes) {
            Pack<T, N> in[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (live && c + j * lanes < packs) in[j] = *reinterpret_cast<const Pack<T, N>*>(from + (c + j * lanes) * N);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (c + j * lanes >= packs) break;
                Pack<O, N> out;
#pragma unroll
                for (int i = 0; i < N; ++i) out.v[i] = rounded<O>(live ? scale * to_float(in[j].v[i]) : 0.0f);
                *reinterpret_cast<Pack<O, N>*>(to + (c + j * lanes) * N) = out;
            }
        }
        // the columns behind the last whole pack
        for (int c = packs * N + part; c < a.width; c += lanes) to[c] = rounded<O>(live ? scale * to_float(from[c]) : 0.0f);
    }
}

bool starts_at(const void* base, long long stride, int bytes, int values) {
    return ((uintptr_t)base & (uintptr_t)(bytes * values - 1)) == 0 && stride % values == 0;
}

template <typename T, typename O, typename K>
int lookup(const fmb_embedding_t& a, cudaStream_t stream) {
    constexpr int kPack = sizeof(T) == 4 || sizeof(O) == 4 ? 4 : 8;
    const bool wide = starts_at(a.source, a.source_stride, sizeof(T), kPack) && starts_at(a.out, a.out_stride, sizeof(O), kPack);
    const int packs = wide ? std::max(1, a.width / kPack) : a.width;
    int lanes = 1;
    while (lanes < 32 && lanes < packs) lanes *= 2;
    const int grid = std::min(ceil_div((long long)a.rows * lanes, 256), 1 << 20);
    if (wide) k_embedding<T, O, K, kPack><<<grid, 256, 0, stream>>>(a, lanes);
    else k_embedding<T, O, K, 1><<<grid, 256, 0, stream>>>(a, lanes);
    FMB_LAUNCH_CHECK();
    return FMB_OK;
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

constexpr int kUnroll = 8;                       // rows on their way

// Columns of a slab: of every lane N side by side (VEC), or N that are 32 apart, where rows do not start at multiples of a pack
template <typename T, bool VEC, int N>
__device__ __forceinline__ int column(int slab, int i) {
    const int lane = threadIdx.x & 31;
    return slab * 32 * N + (VEC ? lane * N + i : lane + 32 * i);
}

template <typename T, bool VEC, int N>
__device__ __forceinline__ void load_columns(const T* __restrict__ row, int slab, int width, float (&x)[N]) {
    const int c0 = column<T, VEC, N>(slab, 0);
    if (VEC && c0 + N <= width) {
        const Pack<T, N> in = *reinterpret_cast<const Pack<T, N>*>(row + c0);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = to_float(in.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = column<T, VEC, N>(slab, i) < width ? to_float(row[column<T, VEC, N>(slab, i)]) : 0.0f;
    }
}

struct Sums {
    fmb_embedding_t a;
    int chunk, chunks, slabs;
    int wide_out;                                // rows of the table start at multiples of 16 bytes
    long long part_stride;                       // floats of a part in scratch: the width, filled up to a multiple of four
    long long sum_ctas;                          // CTAs before those that write zeros
};

// first place whose key is not less than v
__device__ __forceinline__ int lower_bound(const int32_t* __restrict__ keys, int rows, int v) {
    int low = 0, high = rows;
    while (low < high) {
        const int mid = (int)(((unsigned)low + (unsigned)high) >> 1);
        if (__ldg(keys + mid) < v) low = mid + 1; else high = mid;
    }
    return low;
}

__device__ __forceinline__ void write_zeros(const Sums& p) {
    const fmb_embedding_t& a = p.a;
    const int lane = threadIdx.x & 31;
    const int32_t* const keys = (const int32_t*)a.tokens;
    const long long first = ((blockIdx.x - p.sum_ctas) * 8 + (threadIdx.x >> 5)) * 32;
    const int v = (int)min(first + lane, (long long)a.vocabulary);
    bool absent = false;
    if (v < a.vocabulary) {
        const int at = lower_bound(keys, a.rows, v);
        absent = at == a.rows || keys[at] != v;
    }
    for (unsigned left = __ballot_sync(0xffffffffu, absent); left; left &= left - 1) {
        float* const out = (float*)a.out + (first + __ffs(left) - 1) * a.out_stride;
        const int packs = p.wide_out ? a.width / 4 : 0;
        for (int c = lane; c < packs; c += 32) reinterpret_cast<float4*>(out)[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int c = 4 * packs + lane; c < a.width; c += 32) out[c] = 0.0f;
    }
}

template <typename T, bool VEC, int N>
__global__ void __launch_bounds__(256)
k_embedding_sums(Sums p) {
    if (blockIdx.x >= p.sum_ctas) {
        write_zeros(p);
        return;
    }
    const fmb_embedding_t& a = p.a;
    const int32_t* const keys = (const int32_t*)a.tokens;
    const int lane = threadIdx.x & 31;
    const long long unit = blockIdx.x * 8ll + (threadIdx.x >> 5);
    if (unit >= (long long)p.chunks * p.slabs) return;
    const int chunk = (int)(unit / p.slabs), slab = (int)(unit % p.slabs);
    const int begin = chunk * p.chunk, end = min(a.rows, begin + p.chunk);
    const float scale = (float)a.scale;
    // of a run: its key, and whether it began in the chunk before
    int key = __ldg(keys + begin);
    bool before = begin > 0 && __ldg(keys + begin - 1) == key;
    float sum[N];
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i] = 0.0f;

    auto flush = [&](bool after) {
        if (key < 0 || key >= a.vocabulary) return;
        const bool part = before || after;
        float* const out = part ? a.scratch + (2ll * chunk + (before ? 0 : 1)) * p.part_stride : (float*)a.out + key * a.out_stride;
        const bool wide = VEC && (part || p.wide_out);
#pragma unroll
        for (int i0 = 0; i0 < N; i0 += 4) {
            const int c0 = column<T, VEC, N>(slab, i0);
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
                    const int c = column<T, VEC, N>(slab, i);
                    if (c < a.width) out[c] = part ? sum[i] : (a.accumulate ? out[c] : 0.0f) + scale * sum[i];
                }
            }
        }
    };

    for (int p0 = begin; p0 < end; p0 += 32) {
        const int mine = p0 + lane < end ? __ldg(keys + p0 + lane) : a.vocabulary, count = min(32, end - p0);
        int row = p0 + lane < end ? __ldg(a.order + p0 + lane) : -1;
        if (row >= a.rows || mine < 0 || mine >= a.vocabulary) row = -1;
        for (int j0 = 0; j0 < count; j0 += kUnroll) {
            float x[kUnroll][N];
#pragma unroll
            for (int j = 0; j < kUnroll; ++j) {
                const int r = __shfl_sync(0xffffffffu, row, j0 + j);
                if (r >= 0) {
                    load_columns<T, VEC, N>((const T*)a.source + r * a.source_stride, slab, a.width, x[j]);
                } else {
#pragma unroll
                    for (int i = 0; i < N; ++i) x[j][i] = 0.0f;
                }
            }
#pragma unroll
            for (int j = 0; j < kUnroll; ++j) {
                const int next = __shfl_sync(0xffffffffu, mine, j0 + j);
                if (j0 + j < count && next != key) {
                    flush(false);
                    key = next;
                    before = false;
#pragma unroll
                    for (int i = 0; i < N; ++i) sum[i] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < N; ++i) sum[i] += x[j][i];
            }
        }
    }
    flush(end < a.rows && __ldg(keys + end) == key);
}

// The runs that go over the end of the chunk in which they begin: their parts, added in the order of the chunks. A CTA has every
// gridDim.x-th chunk; a run's parts are shared by warps, and slabs of 128 columns by others.
constexpr int kJoinWarps = 32, kJoinList = 64;

__global__ void __launch_bounds__(kJoinWarps * 32)
k_embedding_join(Sums p) {
    __shared__ int list[kJoinList], count;
    __shared__ float4 sums[kJoinWarps][32];
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
            const int parts = (lower_bound(keys, a.rows, key + 1) - 1) / p.chunk - chunk + 1;
            for (int s0 = 0; s0 < slabs; s0 += kJoinWarps / shares) {
                const int slab = s0 + warp / shares, share = warp % shares, c = slab * 128 + 4 * lane;
                float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (c < a.width) {
                    const int from = (int)((long long)parts * share / shares), to = (int)((long long)parts * (share + 1) / shares);
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
                if (share > 0 || c >= a.width) continue;
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

// Rows per chunk: enough chunks for 24 warps on every SM, and as few parts as that leaves; between 16 rows, under which parts cost more
// than they spread, and 256.
int chunk_rows(const fmb_embedding_t& a, int slabs) {
    const long long rows = (long long)a.rows * slabs / (148 * 24) + 1;
    return (int)std::min(256ll, std::max(16ll, (rows + 15) / 16 * 16));
}

bool packed(const fmb_embedding_t& a) {
    return starts_at(a.source, a.source_stride, a.type == FMB_TYPE_F32 ? 4 : 2, a.type == FMB_TYPE_F32 ? 4 : 8);
}

int slabs_of(const fmb_embedding_t& a) { return ceil_div(a.width, a.type == FMB_TYPE_F32 ? 128 : packed(a) ? 256 : 128); }

template <typename T>
int gradient(const fmb_embedding_t& a, cudaStream_t stream) {
    constexpr int kPack = 16 / sizeof(T);
    Sums p;
    p.a = a;
    p.slabs = slabs_of(a);
    p.chunk = chunk_rows(a, p.slabs);
    p.chunks = ceil_div(a.rows, p.chunk);
    p.wide_out = starts_at(a.out, a.out_stride, 4, 4);
    p.part_stride = (a.width + 3) / 4 * 4;
    p.sum_ctas = ceil_div((long long)p.chunks * p.slabs, 8);
    const long long ctas = p.sum_ctas + (a.accumulate ? 0 : ceil_div(a.vocabulary, 256));
    if (ctas > 0) {
        if (packed(a)) k_embedding_sums<T, true, kPack><<<(unsigned)ctas, 256, 0, stream>>>(p);
        else k_embedding_sums<T, false, 4><<<(unsigned)ctas, 256, 0, stream>>>(p);
        FMB_LAUNCH_CHECK();
    }
    if (p.chunks > 1) {
        k_embedding_join<<<std::min(p.chunks, 148), kJoinWarps * 32, 0, stream>>>(p);
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
    const int chunk = chunk_rows(*a, slabs_of(*a));
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
