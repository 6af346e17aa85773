// An expert layer for a few tokens: routing, and the experts' two matrices with the gate between them.
//
//   route:   l = x R; the `top` largest of each token, ties to the lowest number; weights softmax(l) of the chosen, or of all
//   layer:   y[t] = sum_j w[t, j] (silu(x Wg) * (x Wu)) Wd of expert e(t, j)
//
// What bounds the layer is the weights of the experts that are chosen, read once from memory. One launch does it all: units of 32 gate
// columns with the 32 columns they multiply, then units of 64 columns of the second matrix, then units of y, handed out in that order by
// a counter. A unit of the second kind waits for the first ones of its expert, one of y for the second ones of its columns; those were
// handed out before it, so they are done or under way and the wait ends, however few CTAs run at a time.
//
// A unit is 64 columns and 8 or 16 rows over the whole depth, which the eight warps of a CTA share; by sizes (shape_of) several groups of 64
// columns with fewer warps each, or a part of the depth. Each warp has a ring of stages in
// shared memory that asynchronous copies fill, without a barrier between warps; the ring does not run dry between units, since the first
// stages of the next one are asked for before the results of the last are taken out and before a wait for what they multiply. Two
// permutes make pairs along the depth of two rows of the matrix. Columns of the matrix are the MMA's rows, tokens its columns, of which it
// has eight: mma.sync suits that shape (tcgen05 would take 128 columns from shared memory for the same bytes).
//
// Numbers: 16-bit products are exact in fp32. What passes between the products, h, is not rounded to the type of the weights: it is a pair of
// bfloat16 (17 bits, any float32's range) against bfloat16 weights, a pair of tf32 (23 bits) against float16 ones, which are exact in tf32. With
// three bfloat16, all 24 bits, one result of 400 would be rounded otherwise, and results are as far from 64 bits with two as with three
// (1.637e-3 of the norm, their own rounding), at 269 us for 280 (64 tokens, 32 experts of 4,096 x 2,048) and 187 for 218 (35 tokens, 9 of 2,048 x 4,096).
// float32 operands are pairs of tf32 (all but the last of 24 bits), of whose four products the smallest, 2^-22 of the whole, is left out.

#include "early.cuh"
#include "eight.cuh"

#include <algorithm>
#include <type_traits>

namespace fmb {
namespace exp_layer {

namespace {

constexpr int kThreads = 256, kWarps = 8;
constexpr int kUnit = 64;                        // columns of a unit
const float kInfinity = __builtin_huge_valf();
constexpr int kSpins = 1 << 22;                  // polls of a wait, each of 20 ns or more, before a CTA gives up

using eight::rounded;
using eight::to_float;

__device__ __forceinline__ void mma_16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// 16 or 8 bytes, of which the first `bytes` are read and the others zero
__device__ __forceinline__ void copy_16(uint32_t to, const void* from, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_8(uint32_t to, const void* from, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
// whole ones
__device__ __forceinline__ void copy_16(uint32_t to, const void* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory"); }
__device__ __forceinline__ void copy_8(uint32_t to, const void* from) { asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(from) : "memory"); }
__device__ __forceinline__ void copies_end_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint4 load_16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
// --------------------------------------------------------------------------------------------------------------- route


constexpr int kMaxCluster = 8;
constexpr int kRouteChunk = 512;                 // of a CTA's depth, whose values of x lie in shared memory

// eight values as they are in memory, and as floats (one by one where rows are not aligned: with eight.cuh's loads, by words, 64 experts of
// 2,048 in bf16 take a token 4.8 us for 4.5, and 300 at odd distances 75 for 55)
template <typename T> struct Eight { uint32_t v[2 * sizeof(T)]; };

template <typename T>
__device__ __forceinline__ Eight<T> load_eight(const T* __restrict__ at, int live, bool wide) {
    Eight<T> in = {};
    if (wide && live >= 8) {
#pragma unroll
        for (int i = 0; i < 2 * (int)sizeof(T); i += 4) {
            const uint4 four = __ldg(reinterpret_cast<const uint4*>(at) + i / 4);
            in.v[i] = four.x; in.v[i + 1] = four.y; in.v[i + 2] = four.z; in.v[i + 3] = four.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i >= live) break;
            if constexpr (sizeof(T) == 4) in.v[i] = __ldg(reinterpret_cast<const uint32_t*>(at) + i);
            else in.v[i / 2] |= (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(at) + i) << (16 * (i % 2));
        }
    }
    return in;
}

template <typename T>
__device__ __forceinline__ float value(const Eight<T>& in, int i) {
    const uint32_t w = in.v[i * sizeof(T) / 4];
    if constexpr (sizeof(T) == 4) return __uint_as_float(w);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(i % 2 ? w & 0xffff0000u : w << 16);
    else return __half2float(__ushort_as_half((uint16_t)(i % 2 ? w >> 16 : w)));
}

// floats in an order of unsigned numbers; NaN below all
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t bits = __float_as_uint(x + 0.0f);              // (-0 and 0 are equal)
    return x != x ? 0u : bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

// A few tokens. A cluster of eight CTAs for TOKENS tokens: each takes its share of the depth, threads by packs of eight experts and rows of R, which
// all tokens share; then CTA c the choices of token c. A cluster for a token each where there are few (1 token of 2,048, 64 experts: 5.2
// us), for two to eight tokens where they would read much of R one by one.
template <typename T, int TOKENS>
__global__ void __launch_bounds__(kThreads)
k_route(fmb_route_t a, int wide, int rows) {
    constexpr int CLUSTER = kMaxCluster;
    extern __shared__ float sums[];              // [kRouteChunk][TOKENS] values of x; then [TOKENS][rows][packs of eight]
    let_next_come();
    const int first_token = blockIdx.x / CLUSTER * TOKENS, rank = blockIdx.x % CLUSTER, packs = (a.experts + 7) / 8;
    const int pack = threadIdx.x % packs, row = threadIdx.x / packs;
    const int begin = (int)((long long)a.width * rank / CLUSTER), end = (int)((long long)a.width * (rank + 1) / CLUSTER);
    const T* const x = (const T*)a.x + first_token * a.x_stride;
    constexpr int kDeep = sizeof(T) == 4 ? 4 : 8;                 // rows of R on their way
    float sum[TOKENS][8] = {};
    for (int c0 = begin; c0 < end; c0 += kRouteChunk) {
        const int count = min(kRouteChunk, end - c0);
        if (c0 > begin) __syncthreads();
        for (int i = threadIdx.x; i < TOKENS * count; i += kThreads) {
            const int t = i / count, k = i - t * count;
            sums[k * TOKENS + t] = first_token + t < a.tokens ? to_float(x[t * a.x_stride + c0 + k]) : 0.0f;
        }
        __syncthreads();
        if (row >= rows) continue;
        for (int k0 = row; k0 < count; k0 += kDeep * rows) {
            Eight<T> w[kDeep];
#pragma unroll
            for (int j = 0; j < kDeep; ++j) {
                const int k = k0 + j * rows;
                w[j] = load_eight((const T*)a.router + (c0 + k) * a.router_stride + 8 * pack, k < count ? a.experts - 8 * pack : 0, wide);
            }
#pragma unroll
            for (int j = 0; j < kDeep; ++j) {
                const int k = k0 + j * rows;
                if (k >= count) break;
#pragma unroll
                for (int t = 0; t < TOKENS; ++t) {
                    const float v = sums[k * TOKENS + t];
#pragma unroll
                    for (int i = 0; i < 8; ++i) sum[t][i] = fmaf(v, value(w[j], i), sum[t][i]);
                }
            }
        }
    }
    __syncthreads();
    if (row < rows) {
#pragma unroll
        for (int t = 0; t < TOKENS; ++t)
#pragma unroll
            for (int i = 0; i < 8; ++i) sums[(t * rows + row) * packs * 8 + 8 * pack + i] = sum[t][i];
    }
    for (int half = rows / 2; half > 0; half /= 2) {
        __syncthreads();
        const int size = half * packs * 8;
        for (int i = threadIdx.x; i < TOKENS * size; i += kThreads) {
            const int t = TOKENS == 1 ? 0 : i / size, at = t * rows * packs * 8 + i - t * size;
            sums[at] += sums[at + size];
        }
    }
    auto meet = []() { asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory"); };
    meet();
    // An expert's place is the number of those before it (larger logit, or the same and a lower number): each thread counts for its own,
    // which takes one wait where choosing one after the other takes one each. Numbers are made unlike by the expert's.
    __shared__ alignas(16) unsigned long long order[FMB_MAX_GROUPS + 2];
    __shared__ float logits[FMB_MAX_GROUPS], best[FMB_MAX_TOP], warp_total[kWarps];
    static_assert(TOKENS <= CLUSTER, "a CTA for each token's choices");
    const long long token = first_token + rank;
    if (rank < TOKENS && token < a.tokens) {
        for (int e = threadIdx.x; e <= a.experts; e += kThreads) {
            // the CTAs' sums, in their order
            float all = 0.0f;
            if (e < a.experts) {
                const float* const mine = sums + rank * rows * packs * 8 + e;
                const uint32_t here = (uint32_t)__cvta_generic_to_shared(mine);
                float part[CLUSTER];
#pragma unroll
                for (int c = 0; c < CLUSTER; ++c) {
                    uint32_t there;
                    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(here), "r"(c));
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(part[c]) : "r"(there) : "memory");
                }
                all = part[0];
#pragma unroll
                for (int c = 1; c < CLUSTER; ++c) all += part[c];
                logits[e] = all;
            }
            order[e] = e < a.experts ? (unsigned long long)ordered(all) << 32 | (0xffffffffu - e) : 0;
        }
        __syncthreads();
        for (int e = threadIdx.x; e < a.experts; e += kThreads) {
            const unsigned long long mine = order[e];
            int before = 0;
#pragma unroll 4
            for (int f = 0; f < a.experts; f += 2) {
                const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(order + f);
                before += (two.x > mine) + (two.y > mine);
            }
            if (before < a.top) {
                best[before] = logits[e];
                a.chosen[token * a.top + before] = e;
            }
        }
        __syncthreads();
        const float first = best[0];
        float total = 0.0f;
        if (a.normalise) {
            for (int j = 0; j < a.top; ++j) total += expf(best[j] - first);
        } else {
            for (int e = threadIdx.x; e < a.experts; e += kThreads) total += expf(logits[e] - first);
            total = warp_sum(total);
            if ((threadIdx.x & 31) == 0) warp_total[threadIdx.x >> 5] = total;
            __syncthreads();
            total = 0.0f;
            for (int w = 0; w < kWarps; ++w) total += warp_total[w];
        }
        if (threadIdx.x < a.top) a.weights[token * a.top + threadIdx.x] = expf(best[threadIdx.x] - first) / total;
    }
    meet();                                      // shared memory lives until it has been read
}

// Many tokens. A CTA has 16 MT of them and all experts, COLUMNS at a time; a ring of asynchronous copies brings 128 bytes of each row of x and the
// rows of R that they multiply. 16-bit types by matrix instructions, eight warps as MT blocks of 16 tokens by 8 / MT shares of the columns; the sums of a
// stage start at zero and are added to those before with rounding, since the tensor core cuts its sums off. float32 by fused multiply-adds, in which
// all bits count, MT tokens by COLUMNS / 16 columns a thread. Where blocks of tokens are few, the CTAs of a cluster share the depth, and each
// then has every so many of the tokens. A warp chooses for up to four tokens side by side: rounds of the largest of all, which a lane holds a 32nd of.
// 16,384 tokens of 2,048 and 64 experts: bf16 28 us with one choice, 34 with eight (10 for the bytes; issue slots 44 % full, most SMs with two of 256 blocks),
// fp32 137 (60 for the multiply-adds).
template <typename T> constexpr int kRouteDepth = 128 / sizeof(T);

template <int COLUMNS> constexpr int kRouteStages = COLUMNS == 256 ? 3 : 4;
template <int MT, int COLUMNS> constexpr int kRouteRing = kRouteStages<COLUMNS> * 128 * (16 * MT + COLUMNS);
__host__ __device__ constexpr int route_row(int experts) { return (experts + 31) / 32 * 32 + 8; }   // floats of a token's logits, for the banks

__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void load_turned(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}

// 16 bytes of values to shared memory, of which the first `live` values are read and the others zero
template <typename T>
__device__ __forceinline__ void bring_piece(uint32_t to, const T* from, int live, bool wide) {
    constexpr int kValues = 16 / sizeof(T);
    if (wide) {
        copy_16(to, from, (int)sizeof(T) * min(live, kValues));
    } else {
        const Eight<T> in = load_eight(from, min(live, kValues), false);
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(in.v[0]), "r"(in.v[1]), "r"(in.v[2]), "r"(in.v[3]) : "memory");
    }
}

template <typename T, int MT, int COLUMNS, int KEYS>
__global__ void __launch_bounds__(kThreads)
k_route_many(fmb_route_t a, int x_wide, int r_wide, int cluster) {
    constexpr int kTokens = 16 * MT, kRing = kRouteStages<COLUMNS>, kDepth = kRouteDepth<T>, kValues = 16 / sizeof(T);
    constexpr int kXBytes = kTokens * 128, kStageBytes = kXBytes + COLUMNS * 128, kRowBytes = COLUMNS * sizeof(T), kRowPieces = kRowBytes / 16;
    constexpr bool kMatrix = sizeof(T) == 2;
    constexpr bool kOver = KEYS * 32 <= COLUMNS; // the logits take the ring's place
    extern __shared__ __align__(128) uint8_t shared[];
    let_next_come();
    const int rank = blockIdx.x % cluster, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long first_token = (long long)(blockIdx.x / cluster) * kTokens;
    const int tokens = (int)min((long long)kTokens, a.tokens - first_token), stages = (a.width + kDepth - 1) / kDepth;
    const int begin = (int)((long long)stages * rank / cluster), end = (int)((long long)stages * (rank + 1) / cluster);
    const T* const x = (const T*)a.x + first_token * a.x_stride;
    const T* const r = (const T*)a.router;
    float* const logits = reinterpret_cast<float*>(shared + (kOver ? 0 : kRouteRing<MT, COLUMNS>));
    const int row_floats = route_row(a.experts);
    const uint32_t ring = smem_at(shared);

    // of the thread: one piece of every 32nd row of x, and one of every kRowStep-th of R
    constexpr int kRowStep = kThreads / kRowPieces;
    const int x_row = threadIdx.x / 8, x_piece = threadIdx.x % 8, r_row = threadIdx.x / kRowPieces, r_piece = threadIdx.x % kRowPieces;
    const uint32_t x_to = x_row * 128 + (x_piece ^ (x_row & 7)) * 16, r_to = kXBytes + r_row * kRowBytes + (kMatrix ? r_piece ^ (r_row & 7) : r_piece) * 16;
    static_assert((!kMatrix || kRowStep % 8 == 0) && kTokens % 32 == 0, "rows of a thread have one place in their eight");
    const T* x_from[kTokens / 32];
#pragma unroll
    for (int i = 0; i < kTokens / 32; ++i) x_from[i] = x + min(x_row + 32 * i, tokens - 1) * a.x_stride + kValues * x_piece;   // (rows behind the last: anything)
    const bool wide = x_wide && r_wide;

    for (int pass = 0; pass < a.experts; pass += COLUMNS) {
        const int columns = min(COLUMNS, a.experts - pass), r_live = columns - kValues * r_piece, r_bytes = (int)sizeof(T) * min(r_live, kValues);
        const T* const r_from = r + pass + kValues * r_piece + r_row * a.router_stride;
        auto bring = [&](int s, uint32_t to) {
            const int k0 = s * kDepth;
            if (s >= end) {
            } else if (wide && k0 + kDepth <= a.width) {
#pragma unroll
                for (int i = 0; i < kTokens / 32; ++i) copy_16(to + x_to + i * 32 * 128, x_from[i] + k0);
                if (r_live > 0) {
                    const T* from = r_from + k0 * a.router_stride;
#pragma unroll
                    for (int i = 0; i < kDepth / kRowStep; ++i, from += kRowStep * a.router_stride) copy_16(to + r_to + i * kRowStep * kRowBytes, from, r_bytes);
                }
            } else {
                const int x_live = a.width - k0 - kValues * x_piece;
#pragma unroll 1
                for (int i = 0; i < kTokens / 32; ++i) bring_piece(to + x_to + i * 32 * 128, x_live > 0 ? x_from[i] + k0 : x, max(x_live, 0), x_wide);
#pragma unroll 1
                for (int i = 0; i < kDepth / kRowStep; ++i) {
                    const int k = r_row + i * kRowStep, live = k0 + k < a.width ? max(r_live, 0) : 0;
                    bring_piece(to + r_to + i * kRowStep * kRowBytes, live ? r_from + (k0 + i * kRowStep) * a.router_stride : r, live, r_wide);
                }
            }
            copies_end_group();
        };
        for (int s = 0; s < kRing - 1; ++s) bring(begin + s, ring + s * kStageBytes);
        uint32_t slot = 0;
        auto next = [&](int s) {
            copies_wait<kRing - 2>();
            __syncthreads();
            bring(s + kRing - 1, ring + (slot == 0 ? kRing - 1 : slot - 1) * kStageBytes);
            const uint32_t at = ring + slot * kStageBytes;
            slot = slot == kRing - 1 ? 0 : slot + 1;
            return at;
        };
        auto ring_free = [] {                    // for the logits, or for the next pass
            copies_wait<0>();
            __syncthreads();
        };
        if constexpr (kMatrix) {
            constexpr int kShare = COLUMNS * MT / kWarps, kBlocks = kShare / 16;
            const int block = warp % MT, share = warp / MT * kShare;                    // of the warp: tokens, columns of the pass
            const int at_row = lane & 15, at_piece = lane >> 4;
            float sum[2 * kBlocks][4] = {};
            for (int s = begin; s < end; ++s) {
                const uint32_t at = next(s), x_at = at + (16 * block + at_row) * 128, r_at = at + kXBytes + at_row * kRowBytes;
                uint32_t rows[4][4];
#pragma unroll
                for (int k = 0; k < 4; ++k) load_matrices(rows[k], x_at + ((2 * k + at_piece) ^ (at_row & 7)) * 16);
#pragma unroll
                for (int n = 0; n < kBlocks; ++n) {
                    float part[2][4] = {};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        uint32_t b[4];
                        load_turned(b, r_at + k * 16 * kRowBytes + (((share + 16 * n) / 8 + at_piece) ^ (at_row & 7)) * 16);
                        mma_16(part[0], rows[k], b[0], b[1], T());
                        mma_16(part[1], rows[k], b[2], b[3], T());
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum[2 * n][i] += part[0][i], sum[2 * n + 1][i] += part[1][i];
                }
            }
            ring_free();
#pragma unroll
            for (int n = 0; n < 2 * kBlocks; ++n) {
                if (share + 8 * n >= columns) break;
                float* const to = logits + (16 * block + lane / 4) * row_floats + pass + share + 8 * n + lane % 4 * 2;
                *reinterpret_cast<float2*>(to) = make_float2(sum[n][0], sum[n][1]);
                *reinterpret_cast<float2*>(to + 8 * row_floats) = make_float2(sum[n][2], sum[n][3]);
            }
        } else {
            // MT tokens, 16 apart, by groups of four columns, 64 apart
            constexpr int kGroups = COLUMNS / 64;
            const int own = threadIdx.x / 16, four = threadIdx.x % 16;
            float sum[MT][kGroups][4] = {};
            for (int s = begin; s < end; ++s) {
                const uint32_t at = next(s), x_at = at + own * 128, r_at = at + kXBytes + four * 16;
#pragma unroll 2
                for (int k = 0; k < 8; ++k) {
                    uint4 v[MT];
#pragma unroll
                    for (int t = 0; t < MT; ++t) v[t] = load_16(x_at + t * 16 * 128 + (k ^ (own & 7)) * 16);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
#pragma unroll
                        for (int n = 0; n < kGroups; ++n) {
                            const uint4 w = load_16(r_at + (4 * k + i) * kRowBytes + n * 256);
#pragma unroll
                            for (int t = 0; t < MT; ++t) {
                                const float x = __uint_as_float(i == 0 ? v[t].x : i == 1 ? v[t].y : i == 2 ? v[t].z : v[t].w);
                                sum[t][n][0] = fmaf(x, __uint_as_float(w.x), sum[t][n][0]);
                                sum[t][n][1] = fmaf(x, __uint_as_float(w.y), sum[t][n][1]);
                                sum[t][n][2] = fmaf(x, __uint_as_float(w.z), sum[t][n][2]);
                                sum[t][n][3] = fmaf(x, __uint_as_float(w.w), sum[t][n][3]);
                            }
                        }
                    }
                }
            }
            ring_free();
#pragma unroll
            for (int n = 0; n < kGroups; ++n) {
                if (64 * n + 4 * four >= columns) break;
#pragma unroll
                for (int t = 0; t < MT; ++t)
                    *reinterpret_cast<float4*>(logits + (16 * t + own) * row_floats + pass + 64 * n + 4 * four) =
                        make_float4(sum[t][n][0], sum[t][n][1], sum[t][n][2], sum[t][n][3]);
            }
        }
    }
    auto meet = [&]() {
        if (cluster > 1) asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        else __syncthreads();
    };
    meet();
    // keys: an order of numbers above 0, which stands for none: NaN 1
    auto number = [](uint32_t key) {
        const uint32_t bits = key - 1;
        return bits == 0 ? __uint_as_float(0x7fffffffu) : __uint_as_float(bits & 0x80000000u ? bits & 0x7fffffffu : ~bits);
    };
    constexpr int kAtOnce = KEYS > 8 ? 1 : 4;    // tokens of a warp, whose rounds wait side by side
    for (int t0 = warp; rank + t0 * cluster < tokens; t0 += kWarps * kAtOnce) {
        uint32_t key[kAtOnce][KEYS];
        int token[kAtOnce];
#pragma unroll
        for (int b = 0; b < kAtOnce; ++b) {
            token[b] = rank + (t0 + b * kWarps) * cluster;
            const float* const mine = logits + min(token[b], tokens - 1) * row_floats;
#pragma unroll
            for (int i = 0; i < KEYS; ++i) {
                const int e = 32 * i + lane;
                float all = 0.0f;
                if (cluster == 1) {
                    all = e < a.experts ? mine[e] : 0.0f;
                } else if (e < a.experts && token[b] < tokens) {
                    // the CTAs' sums, in their order
                    float part[kMaxCluster];
#pragma unroll
                    for (int c = 0; c < kMaxCluster; ++c) {
                        uint32_t there;
                        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(smem_at(mine + e)), "r"(c < cluster ? c : 0));
                        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(part[c]) : "r"(there) : "memory");
                    }
#pragma unroll
                    for (int c = 0; c < kMaxCluster; ++c) all += c < cluster ? part[c] : 0.0f;
                }
                key[b][i] = e < a.experts ? ordered(all) + 1 : 0;
            }
        }
        float first[kAtOnce], total[kAtOnce], own[kAtOnce];
        int chosen[kAtOnce];
#pragma unroll
        for (int b = 0; b < kAtOnce; ++b) {
            uint32_t best = 0;
#pragma unroll
            for (int i = 0; i < KEYS; ++i) best = max(best, key[b][i]);
            first[b] = number(__reduce_max_sync(0xffffffffu, best));
            total[b] = 0.0f;
            if (a.normalise) continue;
#pragma unroll
            for (int i = 0; i < KEYS; ++i) total[b] += key[b][i] ? expf(number(key[b][i]) - first[b]) : 0.0f;
        }
        for (int j = 0; j < a.top; ++j) {
            uint32_t best[kAtOnce];
            int e[kAtOnce];
#pragma unroll
            for (int b = 0; b < kAtOnce; ++b) {
                best[b] = 0;
#pragma unroll
                for (int i = 0; i < KEYS; ++i) best[b] = max(best[b], key[b][i]);
                best[b] = __reduce_max_sync(0xffffffffu, best[b]);
            }
#pragma unroll
            for (int b = 0; b < kAtOnce; ++b) {
                // the lowest of those that have it
                e[b] = FMB_MAX_GROUPS;
#pragma unroll
                for (int i = KEYS - 1; i >= 0; --i) e[b] = key[b][i] == best[b] ? 32 * i + lane : e[b];
                e[b] = __reduce_min_sync(0xffffffffu, e[b]);
            }
#pragma unroll
            for (int b = 0; b < kAtOnce; ++b) {
#pragma unroll
                for (int i = 0; i < KEYS; ++i) key[b][i] = 32 * i + lane == e[b] ? 0 : key[b][i];
                own[b] = lane == j ? number(best[b]) : own[b];
                chosen[b] = lane == j ? e[b] : chosen[b];
            }
        }
#pragma unroll
        for (int b = 0; b < kAtOnce; ++b) {
            own[b] = lane < a.top ? expf(own[b] - first[b]) : 0.0f;
            total[b] = warp_sum(a.normalise ? own[b] : total[b]);
            if (lane < a.top && token[b] < tokens) {
                const long long to = (first_token + token[b]) * a.top + lane;
                a.chosen[to] = chosen[b];
                a.weights[to] = own[b] / total[b];
            }
        }
    }
    if (cluster > 1) meet();                     // shared memory lives until it has been read
}

// --------------------------------------------------------------------------------------------------------------- layer

__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// x = hi + lo + at most 2^-23 |x|: hi is off by 2^12 steps of x's 24 bits at most, of which lo's 11 hold all but the last. The rest of an infinity is
// NaN (plain_up, plain_down).
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(x - __uint_as_float(hi)));
}

// The same for a weight, of which there are many: in integers, since conversions run at a quarter of the rate (6 tokens, 50 experts of 1,024 x 1,024:
// 74 us by conversions); the rest of an infinity is NaN. What lies below a tf32's bits is cut off, the last bit of 24: 2^-23 |x|, as by rounding.
__device__ __forceinline__ void split_weight(uint32_t x, uint32_t& hi, uint32_t& lo) {
    hi = (x + 0x1000u) & 0xffffe000u;
    lo = __float_as_uint(__uint_as_float(x) - __uint_as_float(hi)) & 0xffffe000u;
}

// What a warp brings at a time, a stage: kDepth rows of the unit's 64 columns and as much of its rows of x or h. For the product a lane has
// kRows neighbouring rows of the depth and eight columns, which are kPieces times 16 bytes, and of block n of the unit's rows one row, kRows
// values of it. Stages lie in shared memory, a ring for each warp, so that no registers wait for them. Copies go along the rows of the
// matrix: lanes that copy what lies side by side (64 bytes that went to lanes four apart came at 3.9 TB/s, and so at 6.9). Rows
// that start at no multiple of 16 bytes (not WIDE) come as the pieces of 16 bytes that they lie in, for each half of the columns one
// more than it fills.
template <typename T, bool WIDE> struct Stage {
    static constexpr int kRows = sizeof(T) == 4 ? 2 : 4, kDepth = 4 * kRows, kPieces = sizeof(T) / 2;
    static constexpr int kHalf = WIDE ? 4 * kPieces : 4 * kPieces + 1;         // pieces of a half
    static constexpr int kMatrixBytes = kDepth * 2 * kHalf * 16, kBytes = kMatrixBytes + 2 * 32 * 16;

    // Where piece c of row kRows quad + j lies: so that the eight lanes that read at a time, of the four quads and pieces of two lanes' columns,
    // find them on different banks.
    __device__ static __forceinline__ int place(int quad, int j, int c) {
        if (WIDE) return (quad * kRows + j) * 2 * kHalf + (c ^ (sizeof(T) == 2 ? 2 * quad : (quad & 1) * 4 + (quad >> 1)));
        return (j * 4 + quad) * 2 * kHalf + c;
    }
};
constexpr int kStages = 3;

__device__ __forceinline__ uint2 load_8(uint32_t at) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
    return v;
}

struct Layer {
    fmb_experts_t a;
    // Of each of the two products: blocks of columns of an expert, groups of 64 columns in a block, which have kWarps / groups warps each for the
    // depth, and units that share the depth of a block
    struct Shape {
        int blocks, log_groups, splits;
        uint32_t inverse;                        // 2^32 / (blocks splits), rounded up
    } up, down;
    int up_share, down_share;                    // stages of a unit
    long long h_stride, part_stride;             // floats of a row: the inner width, or the width, filled up to whole units
    int32_t* control;                            // next unit; of each active expert the blocks that are done; of each block of the second matrix the
                                                 // units; of each block of an active expert's first the units, where they share the depth
    int32_t* lists;                              // number of active experts; active[experts], first[experts + 1], pair[]
    float* h;                                    // [tokens * top]
    float* parts;                                // [down.splits][tokens * top]
    float* up_parts;                             // [up.splits][tokens * top] of h_stride gates and as many they multiply
    void* x;                                     // rows that copies of 8 bytes take: the caller's, or copies of them
    long long x_stride;
};

constexpr int kMaxPairs = FMB_MAX_LAYER_TOKENS * FMB_MAX_TOP;

template <typename T, bool WIDE>
struct Smem {
    alignas(16) uint8_t ring[kWarps][kStages][Stage<T, WIDE>::kBytes];
    float turn[kWarps][kUnit][8];                // results of eight rows on their way out
    uint16_t pair[kMaxPairs];                    // pairs of token and choice, by expert
    uint8_t token[kMaxPairs];
    uint16_t active[FMB_MAX_GROUPS], first[FMB_MAX_GROUPS + 1];
    int ticket, joins;
    volatile int gave_up;
};

struct Unit {
    int up, number, expert, block, part, first, end;
};

template <typename S>
__device__ __forceinline__ Unit unit_of(const Layer& p, const S& s, int ticket, int ups) {
    Unit u;
    u.up = ticket < ups;
    const Layer::Shape& shape = u.up ? p.up : p.down;
    const int t = u.up ? ticket : ticket - ups, per = shape.blocks * shape.splits;
    u.number = per == 1 ? t : (int)__umulhi((uint32_t)t, shape.inverse);
    while (u.number * per > t) --u.number;       // (too large by one where the product is beyond 2^32)
    u.block = t - u.number * per;
    u.part = 0;
    if (shape.splits > 1) {
        u.part = u.block % shape.splits;
        u.block /= shape.splits;
    }
    u.expert = s.active[u.number];
    u.first = s.first[u.number];
    u.end = s.first[u.number + 1];
    return u;
}

// The matrix of a unit as a warp sees it: 32 columns from its first row on, and 32 more `second` bytes behind them; how many bytes of each there
// are; the warp's stages: from `step` to `end`, every hop-th.
struct Matrix {
    const char* at;
    long long second;
    int stride, first_bytes, second_bytes, depth;                              // stride: bytes
    // where this lane's copies of the first stage begin, of kRows rows at once, and whether there is something (not WIDE: the pieces that
    // the halves fill; and the copy of one more piece of each row)
    const char* lane_at;
    bool lane_there;
    int step, end, hop;
};

template <typename T, bool WIDE>
__device__ __forceinline__ Matrix matrix_of(const Layer& p, const Unit& u) {
    const fmb_experts_t& a = p.a;
    constexpr int kSize = sizeof(T);
    Matrix m;
    auto bytes = [](int columns) { return max(0, min(columns, 32)) * kSize; };
    const Layer::Shape& shape = u.up ? p.up : p.down;
    const int warp = threadIdx.x >> 5;
    m.hop = kWarps >> shape.log_groups;
    const int group = (u.block << shape.log_groups) + (warp >> (3 - shape.log_groups));
    if (u.up) {
        m.at = (const char*)((const T*)a.w_up + u.expert * a.up_group_stride + 32 * group);
        m.second = (long long)a.inner * kSize;
        m.first_bytes = m.second_bytes = bytes(a.inner - 32 * group);
        m.stride = (int)a.up_row_stride * kSize;
        m.depth = a.width;
    } else {
        m.at = (const char*)((const T*)a.w_down + u.expert * a.down_group_stride + kUnit * group);
        m.second = 32 * kSize;
        m.first_bytes = bytes(a.width - kUnit * group);
        m.second_bytes = bytes(a.width - kUnit * group - 32);
        m.stride = (int)a.down_row_stride * kSize;
        m.depth = a.inner;
    }
    const int stages = (m.depth + Stage<T, WIDE>::kDepth - 1) / Stage<T, WIDE>::kDepth, share = u.up ? p.up_share : p.down_share;
    m.step = u.part * share + (warp & (m.hop - 1));
    m.end = m.first_bytes > 0 ? min(stages, (u.part + 1) * share) : 0;
    constexpr int kHalf = 4 * Stage<T, WIDE>::kPieces;
    const int lane = threadIdx.x & 31, row = lane / (2 * kHalf), half = lane / kHalf & 1, piece = lane % kHalf;
    m.lane_at = m.at + (long long)m.stride * row + (half ? m.second : 0) + piece * 16;
    m.lane_there = piece * 16 < (half ? m.second_bytes : m.first_bytes);
    return m;
}

// A lane's rows of the unit, up to two, from its first value of the first stage on, and whether they are rows of x
struct Rows {
    const char* at[2];
    bool up;
};

// (Pieces of which a byte belongs to the row are mapped memory, since no piece crosses a page. What they hold beside it, and what is left
// in shared memory where nothing is copied, goes into columns or rows that are not there, which nothing reads.)
template <typename T, bool WIDE>
__device__ __forceinline__ void bring_matrix(const Matrix& m, int step, uint32_t slot) {
    using S = Stage<T, WIDE>;
    const int lane = threadIdx.x & 31, live = m.depth - step * S::kDepth;
    const long long offset = (long long)m.stride * (step * S::kDepth);
    if constexpr (WIDE) {
        // a copy takes kRows rows, those of a quad
        constexpr int kOfRow = 2 * S::kHalf;
        static_assert(kOfRow * S::kRows == 32, "a copy is kRows rows");
        const char* const at = m.lane_at + offset;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t to = slot + S::place(i, lane / kOfRow, lane % kOfRow) * 16;
            const char* const from = at + (long long)m.stride * (i * S::kRows);
            if (live >= S::kDepth) {
                if (m.lane_there) copy_16(to, from);
            } else {
                const bool here = m.lane_there && i * S::kRows + lane / kOfRow < live;
                copy_16(to, here ? from : (const char*)((uintptr_t)m.at & ~(uintptr_t)15), here ? 16 : 0);
            }
        }
    } else {
        // the pieces that a half fills, kRows rows at a time as above, and then the one more of each row
        constexpr int kOfRow = 8 * S::kPieces;
        if (live >= S::kDepth && m.second_bytes == 32 * (int)sizeof(T)) {
            const char* const at = m.lane_at + offset;
            const uint32_t to = slot + S::place(0, lane / kOfRow, lane % kOfRow / (kOfRow / 2) * S::kHalf + lane % (kOfRow / 2)) * 16;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                copy_16(to + S::place(i, 0, 0) * 16, (const char*)((uintptr_t)(at + (long long)m.stride * (i * S::kRows)) & ~(uintptr_t)15));
            const char* const row = m.at + offset + (long long)m.stride * (lane >> 1) + (lane & 1 ? m.second : 0);
            if (lane < 2 * S::kDepth && ((uintptr_t)row & 15))
                copy_16(slot + S::place((lane >> 1) / S::kRows, (lane >> 1) % S::kRows, (lane & 1) * S::kHalf + S::kHalf - 1) * 16,
                        (const char*)((uintptr_t)row & ~(uintptr_t)15) + (S::kHalf - 1) * 16);
            return;
        }
        auto bring = [&](int r, int half, int piece) {
            const char* const row = m.at + offset + (long long)m.stride * r + (half ? m.second : 0);
            const int shift = (int)((uintptr_t)row & 15), bytes = half ? m.second_bytes : m.first_bytes;
            const bool here = r < live && bytes > 0 && piece * 16 < shift + bytes;
            copy_16(slot + S::place(r / S::kRows, r % S::kRows, half * S::kHalf + piece) * 16,
                    here ? row - shift + piece * 16 : (const char*)((uintptr_t)m.at & ~(uintptr_t)15), here ? 16 : 0);
        };
#pragma unroll
        for (int i = 0; i < 4; ++i) bring(i * S::kRows + lane / kOfRow, lane % kOfRow / (kOfRow / 2), lane % (kOfRow / 2));
        if (lane < 2 * S::kDepth) bring(lane >> 1, lane & 1, S::kHalf - 1);
    }
}

// rows of x by kRows values, 8 bytes; of h, which is kept as float32 or, for bfloat16 weights, as four upper halves and then four lower ones
template <typename T, bool WIDE>
__device__ __forceinline__ void bring_rows(const Layer& p, const Rows& r, int depth, int step, uint32_t slot) {
    using S = Stage<T, WIDE>;
    const int lane = threadIdx.x & 31;
    const uint32_t to = slot + S::kMatrixBytes + lane * 16;
    const int offset = step * S::kDepth * (r.up ? (int)sizeof(T) : 4);
    if ((step + 1) * S::kDepth <= depth) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            if (!r.at[n]) continue;
            if (sizeof(T) == 2 && !r.up) copy_16(to + n * 512, r.at[n] + offset);
            else copy_8(to + n * 512, r.at[n] + offset);
        }
        return;
    }
    const int most = depth - step * S::kDepth - S::kRows * (lane & 3);
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const int live = r.at[n] ? max(0, min(S::kRows, most)) : 0;
        const char* const from = live ? r.at[n] + offset : (const char*)p.h;
        if (r.up) copy_8(to + n * 512, from, live * (int)sizeof(T));
        else if (sizeof(T) == 2) copy_16(to + n * 512, from, live ? 16 : 0);
        else copy_8(to + n * 512, from, live ? 8 : 0);
    }
}

// a row's eight values from the pieces they lie in: first by whole words, then by the half
template <typename T>
__device__ __forceinline__ void align_row(uint32_t from, const uint32_t (&v)[sizeof(T) * 2 + 4], uint32_t (&out)[sizeof(T) * 2]) {
    constexpr int kWords = sizeof(T) * 2;
    uint32_t a[kWords + 2], b[kWords + 1];
#pragma unroll
    for (int i = 0; i < kWords + 2; ++i) a[i] = from & 8 ? v[i + 2 < kWords + 4 ? i + 2 : i] : v[i];
#pragma unroll
    for (int i = 0; i < kWords + 1; ++i) b[i] = from & 4 ? a[i + 1] : a[i];
#pragma unroll
    for (int i = 0; i < kWords; ++i) out[i] = sizeof(T) == 2 ? __funnelshift_r(b[i], b[i + 1], (from & 2) * 8) : b[i];
}

// The stage's product, for rows of x (up) or h, one block of eight rows or two: branches that the whole warp takes, in one body, since with
// a body for each case the code of a unit's end was waited for longer than it took. Matrix columns are the MMA's rows, in the order of
// the lanes' eight: acc[i][n] has columns 2 i and 2 i + 1.
template <typename T, bool WIDE>
__device__ __forceinline__ void multiply(float (&acc)[4][2][4], const Matrix& m, int step, uint32_t slot, bool up, bool two_blocks) {
    using S = Stage<T, WIDE>;
    constexpr int kWords = sizeof(T) * 2;
    const int lane = threadIdx.x & 31, g = lane >> 2, quad = lane & 3;
    uint32_t w[S::kRows][kWords];
#pragma unroll
    for (int j = 0; j < S::kRows; ++j) {
        if (WIDE) {
#pragma unroll
            for (int i = 0; i < S::kPieces; ++i) {
                const uint4 v = load_16(slot + S::place(quad, j, g * S::kPieces + i) * 16);
                w[j][4 * i] = v.x; w[j][4 * i + 1] = v.y; w[j][4 * i + 2] = v.z; w[j][4 * i + 3] = v.w;
            }
        } else {
            uint32_t raw[kWords + 4];
#pragma unroll
            for (int i = 0; i <= S::kPieces; ++i) {
                const uint4 v = load_16(slot + S::place(quad, j, (g >> 2) * S::kHalf + (g & 3) * S::kPieces + i) * 16);
                raw[4 * i] = v.x; raw[4 * i + 1] = v.y; raw[4 * i + 2] = v.z; raw[4 * i + 3] = v.w;
            }
            align_row<T>(((uint32_t)(uintptr_t)m.at + (g >> 2 ? (uint32_t)m.second : 0u) + (uint32_t)m.stride * (step * S::kDepth + S::kRows * quad + j)) & 15, raw, w[j]);
        }
    }
    const uint32_t rows = slot + S::kMatrixBytes + lane * 16;
    if (sizeof(T) == 2 && (up || std::is_same<T, __nv_bfloat16>::value)) {
        if constexpr (sizeof(T) == 2) {
            uint32_t a[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i][0] = __byte_perm(w[0][i], w[1][i], 0x5410);
                a[i][1] = __byte_perm(w[0][i], w[1][i], 0x7632);
                a[i][2] = __byte_perm(w[2][i], w[3][i], 0x5410);
                a[i][3] = __byte_perm(w[2][i], w[3][i], 0x7632);
            }
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                if (n && !two_blocks) break;
                const uint4 b = load_16(rows + n * 512);          // (of x the first half)
                if (!up) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) mma_16(acc[i][n], a[i], b.z, b.w, T());
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) mma_16(acc[i][n], a[i], b.x, b.y, T());
            }
        }
    } else {
        // float32 values as pairs of tf32, float16 weights as they are
        auto add = [&](auto blocks) {
            constexpr int NB = decltype(blocks)::value;
            uint32_t hi[NB][S::kRows], lo[NB][S::kRows];
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                float b[S::kRows];
                if constexpr (S::kRows == 4) {
                    const uint4 v = load_16(rows + n * 512);
                    b[0] = __uint_as_float(v.x); b[1] = __uint_as_float(v.y); b[2] = __uint_as_float(v.z); b[3] = __uint_as_float(v.w);
                } else {
                    const uint2 v = load_8(rows + n * 512);
                    b[0] = __uint_as_float(v.x); b[1] = __uint_as_float(v.y);
                }
#pragma unroll
                for (int q = 0; q < S::kRows; ++q) split_tf32(b[q], hi[n][q], lo[n][q]);
            }
#pragma unroll
            for (int s = 0; s < S::kRows / 2; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t a[4], rest[4];
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        if constexpr (sizeof(T) == 2) {
                            const float2 two = __half22float2(*reinterpret_cast<const __half2*>(&w[2 * s + q][i]));
                            a[2 * q] = __float_as_uint(two.x);
                            a[2 * q + 1] = __float_as_uint(two.y);
                        } else {
                            split_weight(w[2 * s + q][2 * i], a[2 * q], rest[2 * q]);
                            split_weight(w[2 * s + q][2 * i + 1], a[2 * q + 1], rest[2 * q + 1]);
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NB; ++n) {
                        if constexpr (sizeof(T) == 4) {
                            // The tensor core cuts its sums off, which adds up along the depth (float32 results were 8e-6 off at a depth
                            // of 4,096): each stage's sum begins at zero and is added with rounding.
                            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                            mma_tf32(sum, a, lo[n][2 * s], lo[n][2 * s + 1]);
                            mma_tf32(sum, rest, hi[n][2 * s], hi[n][2 * s + 1]);
                            mma_tf32(sum, a, hi[n][2 * s], hi[n][2 * s + 1]);
#pragma unroll
                            for (int q = 0; q < 4; ++q) acc[i][n][q] += sum[q];
                        } else {
                            mma_tf32(acc[i][n], a, lo[n][2 * s], lo[n][2 * s + 1]);
                            mma_tf32(acc[i][n], a, hi[n][2 * s], hi[n][2 * s + 1]);
                        }
                    }
                }
        };
        if (two_blocks) add(std::integral_constant<int, 2>());
        else add(std::integral_constant<int, 1>());
    }
}

// The CTA's coming unit of the second matrix into the L2, so that memory does not wait for the first products with it: lines of
// 128 bytes, up to 1,024 rows (at F = 1,024 the units of all CTAs are 38 MB).
__device__ __forceinline__ void prefetch_unit(const Matrix& m) {
    if (m.first_bytes == 0) return;
    const int rows = min(m.depth, 1024);
    for (int k = ((threadIdx.x >> 5) & (m.hop - 1)) * 32 + (threadIdx.x & 31); k < rows; k += m.hop * 32) {
        const char* const at = m.at + (long long)m.stride * k;
        asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
        const char* const last = at + (m.second_bytes > 0 ? m.second + m.second_bytes : m.first_bytes) - 1;
        if (((uintptr_t)last ^ (uintptr_t)at) >> 7) asm volatile("prefetch.global.L2 [%0];" ::"l"(last));
    }
}

// one more at a counter, behind what this CTA has written before its last barrier
__device__ __forceinline__ void add_release(int32_t* at) { asm volatile("red.release.gpu.global.add.s32 [%0], 1;" ::"l"(at) : "memory"); }
__device__ __forceinline__ int add_acquire_release(int32_t* at) {
    int before;
    asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(before) : "l"(at) : "memory");
    return before;
}

__device__ __forceinline__ int load_relaxed(const int32_t* at) {
    int v;
    asm volatile("ld.relaxed.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(at) : "memory");
    return v;
}

__device__ __forceinline__ int load_acquire(const int32_t* at) {
    int v;
    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(at) : "memory");
    return v;
}

// The state of a warp's ring between the units: the place of the next stage, and what has been asked for of the coming unit.
struct Ring {
    uint32_t base;
    int place;

    template <int BYTES> __device__ __forceinline__ uint32_t slot(int ahead) const {
        const int at = place + ahead;
        return base + (at >= kStages ? at - kStages : at) * BYTES;
    }
};

template <typename T, bool WIDE>
__device__ __forceinline__ Rows rows_of(const Layer& p, const Smem<T, WIDE>& s, const Unit& u, int first) {
    Rows r;
    const int g = (threadIdx.x & 31) >> 2;
    r.up = u.up;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const int at = first + 8 * n + g;
        r.at[n] = nullptr;
        if (at >= u.end) continue;
        const int k = Stage<T, WIDE>::kRows * (threadIdx.x & 3);
        r.at[n] = u.up ? (const char*)((const T*)p.x + s.token[at] * p.x_stride + k) : (const char*)(p.h + s.pair[at] * p.h_stride + k);
    }
    return r;
}

// one warp's first stages of a unit, the matrix or the rows or both; a group of copies each
template <typename T, bool WIDE>
__device__ __forceinline__ void begin(const Layer& p, const Ring& ring, const Matrix& m, const Rows& r, bool matrix, bool rows) {
    using S = Stage<T, WIDE>;
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
        const int step = m.step + i * m.hop;
        const uint32_t slot = ring.template slot<S::kBytes>(i);
        // (nothing is asked for past the end: it would not be waited for before its place is filled again)
        if (step < m.end) {
            if (matrix) bring_matrix<T, WIDE>(m, step, slot);
            if (rows) bring_rows<T, WIDE>(p, r, m.depth, step, slot);
        }
        copies_end_group();
    }
}

// The sums over the depth of a unit's 64 columns and up to 16 rows. All of the first stages have been asked for; `all`: only the wait
// for every copy covers them.
template <typename T, bool WIDE>
__device__ __forceinline__ void product(const Layer& p, Ring& ring, const Matrix& m, const Rows& r, bool all, bool two_blocks, float (&acc)[4][2][4]) {
    using S = Stage<T, WIDE>;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[i][n][q] = 0.0f;
    if (all) copies_wait<0>();
    for (int step = m.step; step < m.end; step += m.hop) {
        copies_wait<kStages - 2>();
        __syncwarp();                            // every lane's copies of this stage are here, and the stage before has been read
        const uint32_t next = ring.template slot<S::kBytes>(kStages - 1);
        const int coming = step + (kStages - 1) * m.hop;
        if (coming < m.end) {
            bring_matrix<T, WIDE>(m, coming, next);
            bring_rows<T, WIDE>(p, r, m.depth, coming, next);
        }
        copies_end_group();
        multiply<T, WIDE>(acc, m, step, ring.template slot<S::kBytes>(0), r.up, two_blocks);
        ring.place = ring.place + 1 == kStages ? 0 : ring.place + 1;
    }
    __syncwarp();
}

// Block n of the warps' sums on its way out: column 8 g + j at place 8 j + g, so that the lanes' stores and loads fall on different banks
__device__ __forceinline__ void turn_in(float (&turn)[kWarps][kUnit][8], const float (&acc)[4][2][4], int n) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int b = 0; b < 2; ++b)
            *reinterpret_cast<float2*>(&turn[warp][(2 * i + b) * 8 + (lane >> 2)][2 * (lane & 3)]) =
                n == 0 ? make_float2(acc[i][0][2 * b], acc[i][0][2 * b + 1]) : make_float2(acc[i][1][2 * b], acc[i][1][2 * b + 1]);
}

template <typename T>
__device__ __forceinline__ void put_h(const Layer& p, int pair, int column, float gate, float up) {
    const float h = column < p.a.inner ? gate / (1.0f + expf(-gate)) * up : 0.0f;
    float* const to = p.h + pair * p.h_stride;
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        // (what would be rounded past bfloat16's largest number is cut off instead)
        const __nv_bfloat16 hi = fabsf(h) <= 3.3e38f ? __float2bfloat16_rn(h) : __float2bfloat16_rz(h);
        const float rest = fabsf(h) < kInfinity ? h - __bfloat162float(hi) : 0.0f;
        __nv_bfloat16* const four = (__nv_bfloat16*)(to + (column & ~3));
        four[column & 3] = hi;
        four[4 + (column & 3)] = __float2bfloat16_rn(rest);
    } else {
        to[column] = h;
    }
}

// h as put_h has kept it
template <typename T>
__device__ __forceinline__ float get_h(const float* h, int column) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const uint16_t* const four = (const uint16_t*)(h + (column & ~3));
        return __uint_as_float((uint32_t)__ldcg(four + (column & 3)) << 16) + __uint_as_float((uint32_t)__ldcg(four + 4 + (column & 3)) << 16);
    } else {
        return __ldcg(h + column);
    }
}

// Where operands are split in parts, an infinite one is multiplied with another's zero rest, and one near the largest number is rounded to
// infinity. Such a sum is not finite, so what is not is asked of a plain product, by a thread alone: slow, and not met where numbers are (it ends
// with the first NaN: 6 tokens, 50 experts of 1,024 x 1,024 in fp32 55 us, with a token of NaN 74, with one infinite x 911).
// In the first product those are sums of float32 (x and weights of 16 bits are multiplied as they are), by the CTA whose unit they are, after it;
template <typename T, bool WIDE>
__device__ __noinline__ void plain_up(const Layer& p, const Smem<T, WIDE>& s, const Unit& u) {
    const int columns = 32 << p.up.log_groups, share = p.up_share * Stage<T, WIDE>::kDepth, begin = u.part * share, end = min(p.a.width, begin + share);
    const long long pairs = (long long)p.a.tokens * p.a.top, stride = p.a.up_row_stride;
    for (int i = threadIdx.x; i < (u.end - u.first) * columns; i += kThreads) {
        const int at = u.first + i / columns, pair = s.pair[at], column = u.block * columns + i % columns;
        if (column >= p.a.inner) continue;
        float* const parts = p.up_parts + (u.part * pairs + pair) * 2 * p.h_stride + column;
        const bool shared = p.up.splits > 1;
        if (fabsf(shared ? parts[0] + parts[p.h_stride] : p.h[pair * p.h_stride + column]) < kInfinity) continue;
        const T* const x = (const T*)p.x + s.token[at] * p.x_stride;
        const T* const w = (const T*)p.a.w_up + u.expert * p.a.up_group_stride + column;
        float gate = 0.0f, up = 0.0f;
#pragma unroll 4
        for (int k = begin; k < end; ++k) {
            gate = fmaf(to_float(x[k]), to_float(w[k * stride]), gate);
            up = fmaf(to_float(x[k]), to_float(w[k * stride + p.a.inner]), up);
            if (gate != gate && up != up) break;
        }
        if (shared) parts[0] = gate, parts[p.h_stride] = up;
        else put_h<T>(p, pair, column, gate, up);
    }
}

// in the second all, found by their weighted sum: a column of y with what is not finite of its parts anew.
template <typename T>
__device__ __noinline__ float plain_down(const Layer& p, int t, int column) {
    const fmb_experts_t& a = p.a;
    const long long pairs = (long long)a.tokens * a.top;
    float sum = 0.0f;
    for (int j = 0; j < a.top; ++j) {
        const long long pair = (long long)t * a.top + j;
        const int e = __ldcg(a.chosen + pair);
        if (e < 0 || e >= a.experts) continue;
        float v = 0.0f;
        for (int part = 0; part < p.down.splits; ++part) v += __ldcg(p.parts + (part * pairs + pair) * p.part_stride + column);
        if (!(fabsf(v) < kInfinity)) {
            const T* const w = (const T*)a.w_down + e * a.down_group_stride + column;
            const float* const h = p.h + pair * p.h_stride;
            v = 0.0f;
#pragma unroll 4
            for (int k = 0; k < a.inner && v == v; ++k) v = fmaf(get_h<T>(h, k), to_float(w[k * a.down_row_stride]), v);
        }
        sum += __ldcg(a.weights + pair) * v;
    }
    return sum;
}

// Lane l of warp j takes columns 8 (l / 8) + j and that + 32 of row l % 8 out, of each group of 64: the gate's result for h, or the two columns
// of a pair's part. `finite`: whether this thread's sums of float32 for h still are.
template <typename T, bool WIDE>
__device__ __forceinline__ void turn_out(const Layer& p, const Smem<T, WIDE>& s, const Unit& u, int first, bool& finite) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, at = first + (lane & 7);
    const Layer::Shape& shape = u.up ? p.up : p.down;
    const int warps = kWarps >> shape.log_groups;
    const long long pairs = (long long)p.a.tokens * p.a.top;
    for (int q = 0; q < 1 << shape.log_groups; ++q) {
        float low = 0.0f, high = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w >= warps) break;
            low += s.turn[q * warps + w][8 * warp + (lane >> 3)][lane & 7];
            high += s.turn[q * warps + w][8 * warp + 4 + (lane >> 3)][lane & 7];
        }
        if (at >= u.end) continue;
        const int group = (u.block << shape.log_groups) + q, place = 8 * (lane >> 3) + warp, pair = s.pair[at];
        if (!u.up) {
            if (kUnit * group >= p.part_stride) continue;
            float* const to = p.parts + (u.part * pairs + pair) * p.part_stride + kUnit * group + place;
            to[0] = low;
            to[32] = high;
        } else if (32 * group < p.h_stride) {
            if (sizeof(T) == 4) finite &= fabsf(low + high) < kInfinity || 32 * group + place >= p.a.inner;
            if (shape.splits > 1) {
                float* const to = p.up_parts + (u.part * pairs + pair) * 2 * p.h_stride + 32 * group + place;
                to[0] = low;
                to[p.h_stride] = high;
            } else {
                put_h<T>(p, pair, 32 * group + place, low, high);
            }
        }
    }
}

// h of a block whose depth units have shared, by the one that was done last
template <typename T, bool WIDE>
__device__ __noinline__ void join_up(const Layer& p, const Smem<T, WIDE>& s, const Unit& u) {
    const int columns = 32 << p.up.log_groups, first = u.block * columns;
    const long long pairs = (long long)p.a.tokens * p.a.top;
    for (int i = threadIdx.x; i < (u.end - u.first) * columns; i += kThreads) {
        const int pair = s.pair[u.first + i / columns], column = first + i % columns;
        if (column >= p.h_stride) continue;
        float gate = 0.0f, up = 0.0f;
#pragma unroll 4
        for (int part = 0; part < p.up.splits; ++part) {
            const float* const from = p.up_parts + (part * pairs + pair) * 2 * p.h_stride + column;
            gate += __ldcg(from);
            up += __ldcg(from + p.h_stride);
        }
        put_h<T>(p, pair, column, gate, up);
    }
}

// y of 64 columns and kCombined tokens: what the experts of each token have given, in the order of its choices. Four columns a thread. The
// weights are asked for before the wait for the parts (`await`).
constexpr int kCombined = kThreads / 16;

template <typename T, typename F>
__device__ __forceinline__ void combine(const Layer& p, int group, int tokens, F await) {
    const fmb_experts_t& a = p.a;
    const long long pairs = (long long)a.tokens * a.top;
    const int c = kUnit * group + 4 * (threadIdx.x & 15), t = tokens * kCombined + (threadIdx.x >> 4);
    const bool exists = c < a.width && t < a.tokens;
    float w[FMB_MAX_TOP];
    unsigned live = 0;                           // choices that are experts: of the others nothing has been written
#pragma unroll
    for (int j = 0; j < FMB_MAX_TOP; ++j) {
        const bool there = exists && j < a.top;
        const int e = there ? __ldcg(a.chosen + t * a.top + j) : -1;
        w[j] = there ? __ldcg(a.weights + t * a.top + j) : 0.0f;
        if (e >= 0 && e < a.experts) live |= 1u << j;
    }
    await();
    if (!exists) return;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int j0 = 0; j0 < FMB_MAX_TOP; j0 += 8) {
        if (j0 >= a.top) break;
        float4 v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float* const from = p.parts + (t * a.top + j0 + j) * p.part_stride + c;
            const bool there = live >> (j0 + j) & 1;
            v[j] = there ? __ldcg(reinterpret_cast<const float4*>(from)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (int part = 1; part < p.down.splits && there; ++part) {
                const float4 more = __ldcg(reinterpret_cast<const float4*>(from + part * pairs * p.part_stride));
                v[j].x += more.x; v[j].y += more.y; v[j].z += more.z; v[j].w += more.w;
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (!(live >> (j0 + j) & 1)) continue;
            sum.x += w[j0 + j] * v[j].x;
            sum.y += w[j0 + j] * v[j].y;
            sum.z += w[j0 + j] * v[j].z;
            sum.w += w[j0 + j] * v[j].w;
        }
    }
    T* const y = (T*)a.y + t * a.y_stride + c;
    float out[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (c + i >= a.width) break;
        if (!(fabsf(out[i]) < kInfinity)) out[i] = plain_down<T>(p, t, c + i);
        y[i] = rounded<T>(out[i]);
    }
}

// Which pairs belong to which expert, and which experts have any; the counters of the next launch become zero. Pairs of one expert stand in
// any order: their results do not depend on it. A thread for every expert and every two pairs. The CTAs behind the first copy rows of x, where those do not begin at multiples
// of 8 bytes.
template <typename T>
__global__ void __launch_bounds__(1024)
k_list_pairs(Layer p, int control, void* packed) {
    const fmb_experts_t& a = p.a;
    let_next_come();
    kernels_before(p.a.x, p.a.chosen);           // what the rows and the choices come from
    if (blockIdx.x > 0) {
        const T* const from = (const T*)a.x + (blockIdx.x - 1) * a.x_stride;
        T* const to = (T*)packed + (blockIdx.x - 1) * p.x_stride;
        for (int c = threadIdx.x; c < p.x_stride; c += blockDim.x) to[c] = c < a.width ? from[c] : T(0.0f);
        return;
    }
    __shared__ int start[FMB_MAX_GROUPS];
    __shared__ int warp_total[2][32];
    const int experts = a.experts, pairs = a.tokens * a.top, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = threadIdx.x;
    int32_t* const active = p.lists + 1;
    int32_t* const first = active + experts;
    int32_t* const pair = first + experts + 1;
    for (int i = threadIdx.x; i < control; i += blockDim.x) p.control[i] = 0;
    start[e] = 0;
    __syncthreads();
    int chosen[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int i = threadIdx.x + blockDim.x * q;
        chosen[q] = i < pairs ? __ldg(a.chosen + i) : -1;
        if (chosen[q] >= experts) chosen[q] = -1;
        if (chosen[q] >= 0) atomicAdd(start + chosen[q], 1);
    }
    __syncthreads();
    const int count = start[e];
    int sums = count, somes = count > 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, sums, o), y = __shfl_up_sync(0xffffffffu, somes, o);
        if (lane >= o) sums += x, somes += y;
    }
    if (lane == 31) warp_total[0][warp] = sums, warp_total[1][warp] = somes;
    __syncthreads();
    int before = lane < warp ? warp_total[0][lane] : 0, number = lane < warp ? warp_total[1][lane] : 0;
    before = warp_sum(before);
    number = warp_sum(number);
    const int begin = before + sums - count, place = number + somes - (count > 0);
    start[e] = begin;
    if (count > 0) {
        active[place] = e;
        first[place] = begin;
    }
    if (e == blockDim.x - 1) {
        first[place + (count > 0)] = begin + count;
        p.lists[0] = place + (count > 0);
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 2; ++q)
        if (chosen[q] >= 0) pair[atomicAdd(start + chosen[q], 1)] = threadIdx.x + blockDim.x * q;
}

template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads, 2)
k_experts(const __grid_constant__ Layer p) {
    extern __shared__ __align__(16) uint8_t smem[];
    Smem<T, WIDE>& s = *reinterpret_cast<Smem<T, WIDE>*>(smem);
    const fmb_experts_t& a = p.a;
    int32_t* const next = p.control;
    int32_t* const done = p.control + 1;
    int32_t* const columns = done + a.experts;
    const int32_t* lists = p.lists;
    kernels_before(lists);
    if (threadIdx.x == 0) {
        s.ticket = atomicAdd(next, 1);
        s.gave_up = 0;
    }
    // (the lists' places, whether in use or not: their numbers need not be waited for)
    const int actives = __ldg(lists), most = min(a.experts, a.tokens * a.top);
    for (int i = threadIdx.x; i <= most; i += kThreads) {
        if (i < most) s.active[i] = (uint16_t)__ldg(lists + 1 + i);
        s.first[i] = (uint16_t)__ldg(lists + 1 + a.experts + i);
    }
    for (int i = threadIdx.x; i < a.tokens * a.top; i += kThreads) {
        const uint32_t pair = (uint32_t)__ldg(lists + 2 + 2 * a.experts + i);
        s.pair[i] = (uint16_t)pair;
        s.token[i] = (uint8_t)(pair / a.top);
    }
    __syncthreads();
    if (actives == 0) {                          // no expert is one
        for (long long i = blockIdx.x * (long long)kThreads + threadIdx.x; i < (long long)a.tokens * a.width; i += (long long)gridDim.x * kThreads)
            ((T*)a.y)[i / a.width * a.y_stride + i % a.width] = T(0.0f);
        return;
    }
    // three kinds of units, of which each waits for ones of the kind before: h, the parts of y, and y
    const int ups = actives * p.up.blocks * p.up.splits, downs = ups + actives * p.down.blocks * p.down.splits;
    const int groups = (a.width + kUnit - 1) / kUnit, units = downs + groups * ((a.tokens + kCombined - 1) / kCombined);
    int32_t* const shared = columns + p.down.blocks;
    // Thread 0 waits for a counter, with a limit, after which all waits end at once and the results are said to be none; the others wait for it
    // (2,048 warps that ask for the same eight counters hold up those that count)
    auto await = [&](const int32_t* counter, int value) {
        if (threadIdx.x == 0) {
            int spins = 0;
            while (load_relaxed(counter) < value && !s.gave_up)
                if (++spins < kSpins) __nanosleep(20);
                else s.gave_up = 1;
            (void)load_acquire(counter);
            if (s.gave_up && a.status) atomicOr(a.status, (uint32_t)FMB_STATUS_TENSOR_TIMEOUT);
        }
        __syncthreads();
    };
    int ticket = s.ticket;
    Unit u;
    Matrix m;
    Rows r;
    Ring ring = {smem_at(s.ring[threadIdx.x >> 5]), 0};
    bool ready = false, turning = false;         // ready: what the unit's rows are has been written
    // the ticket's unit, if it is one of a product, and its first stages
    auto go_on = [&]() {
        if (ticket >= downs) return;
        u = unit_of(p, s, ticket, ups);
        m = matrix_of<T, WIDE>(p, u);
        r = rows_of<T, WIDE>(p, s, u, u.first);
        ready = u.up;
        begin<T, WIDE>(p, ring, m, r, true, ready);
        if (turning) prefetch_unit(m);
    };
    go_on();
    while (ticket < downs) {
        bool all = false;
        if (!ready) {
            await(done + u.number, p.up.blocks);
            begin<T, WIDE>(p, ring, m, r, false, true);
            all = true;
        }
        // The unit after this one: asked for now, when this one no longer waits for others, and needed at its end.
        const int ahead = threadIdx.x == 0 ? atomicAdd(next, 1) : 0;
        const Unit v = u;
        bool finite = true;
        for (int at = v.first; at < v.end; at += 16) {
            const bool last = at + 16 >= v.end, two_blocks = v.end - at > 8;
            float acc[4][2][4];
            product<T, WIDE>(p, ring, m, r, all, two_blocks, acc);
            all = false;
            if (last && threadIdx.x == 0) s.ticket = ahead;
            turn_in(s.turn, acc, 0);
            __syncthreads();
            // Copies are on their way while results are taken out. Only where the next unit waits for first products, this one's are given
            // to the others first: all CTAs come to that point at the same time.
            if (last) {
                ticket = s.ticket;
                turning = v.up && ticket >= ups;
                if (!turning) go_on();
            } else {
                r = rows_of<T, WIDE>(p, s, v, at + 16);
                begin<T, WIDE>(p, ring, m, r, true, true);
            }
            turn_out<T, WIDE>(p, s, v, at, finite);
            __syncthreads();                     // the sums have been read, and what they gave is written
            if (two_blocks) {
                turn_in(s.turn, acc, 1);
                __syncthreads();
                turn_out<T, WIDE>(p, s, v, at + 8, finite);
                __syncthreads();
            }
        }
        if (sizeof(T) == 4 && v.up && !__syncthreads_and(finite)) {
            plain_up<T, WIDE>(p, s, v);
            __syncthreads();
        }
        bool tells = true;                       // thread 0, while its CTA goes on
        if (v.up && p.up.splits > 1) {
            if (threadIdx.x == 0) s.joins = add_acquire_release(shared + v.number * p.up.blocks + v.block) == p.up.splits - 1;
            __syncthreads();
            tells = s.joins;
            if (tells) join_up<T, WIDE>(p, s, v);
            __syncthreads();
        }
        if (threadIdx.x == 0 && tells) add_release(v.up ? done + v.number : columns + v.block);
        if (turning) go_on();
    }
    while (ticket < units) {
        const int group = (ticket - downs) % groups, tokens = (ticket - downs) / groups;
        // (the barrier of the wait: the ticket has been read)
        combine<T>(p, group, tokens, [&]() { await(columns + (group >> p.down.log_groups), actives * p.down.splits); });
        if (threadIdx.x == 0) s.ticket = atomicAdd(next, 1);
        __syncthreads();
        ticket = s.ticket;
    }
}

long long up_to(long long n, long long step) { return (n + step - 1) / step * step; }

// How a product with `columns` (32 or 64 a group) and `depth` is cut for the experts that tokens choose at most.
Layer::Shape shape_of(int experts, int columns, int of_group, int depth, int stage_depth) {
    constexpr int kCtas = 2 * 148;
    Layer::Shape s;
    const int stages = ceil_div(depth, stage_depth);
    s.log_groups = 0;
    s.splits = 1;
    while (s.log_groups < 3 && stages << s.log_groups < 8 * kWarps && (long long)experts * ceil_div(columns, of_group << (s.log_groups + 1)) >= 2 * kCtas) ++s.log_groups;
    s.blocks = ceil_div(columns, of_group << s.log_groups);
    const long long units = (long long)experts * s.blocks;
    if (2 * units <= kCtas) s.splits = (int)std::max<long long>(1, std::min<long long>({8, kCtas / units, stages / (2 * kWarps)}));
    s.inverse = (uint32_t)(((1ull << 32) + s.blocks * s.splits - 1) / (s.blocks * s.splits));
    return s;
}

struct Sizes {
    Layer::Shape up, down;
    long long control, lists, h, parts, up_parts, x;              // in floats
    long long h_stride, part_stride, x_stride;
};

Sizes sizes_of(const fmb_experts_t& a) {
    Sizes s;
    const long long pairs = (long long)a.tokens * a.top;
    const int experts = (int)std::min<long long>(a.experts, pairs), stage = a.type == FMB_TYPE_F32 ? Stage<float, true>::kDepth : Stage<__half, true>::kDepth;
    s.up = shape_of(experts, a.inner, 32, a.width, stage);
    s.down = shape_of(experts, a.width, kUnit, a.inner, stage);
    s.control = up_to(1 + a.experts + s.down.blocks + (s.up.splits > 1 ? (long long)experts * s.up.blocks : 0), 64);
    s.lists = up_to(2 + 2 * a.experts + pairs, 64);
    s.h_stride = up_to(a.inner, 32);
    s.part_stride = up_to(a.width, kUnit);
    s.h = pairs * s.h_stride;
    s.parts = s.down.splits * pairs * s.part_stride;
    s.up_parts = s.up.splits > 1 ? s.up.splits * pairs * 2 * s.h_stride : 0;
    s.x_stride = up_to(a.width, 8);
    s.x = a.tokens * s.x_stride;
    return s;
}

// whether the rows of a matrix begin at multiples of `unit` bytes
bool begin_at(const void* base, long long stride, int rows, int bytes, int unit) {
    return (uintptr_t)base % unit == 0 && (rows <= 1 || stride * bytes % unit == 0);
}

template <typename T>
int layer(const fmb_experts_t& a, cudaStream_t stream) {
    const Sizes size = sizes_of(a);
    const int b = sizeof(T);
    Layer p;
    p.a = a;
    p.control = (int32_t*)a.scratch;
    p.lists = p.control + size.control;
    p.h = a.scratch + size.control + size.lists;
    p.parts = p.h + size.h;
    p.up_parts = p.parts + size.parts;
    void* const packed = p.up_parts + size.up_parts;
    p.h_stride = size.h_stride;
    p.part_stride = size.part_stride;
    p.up = size.up;
    p.down = size.down;
    const int stage = sizeof(T) == 4 ? Stage<float, true>::kDepth : Stage<__half, true>::kDepth;
    p.up_share = ceil_div(ceil_div(a.width, stage), p.up.splits);
    p.down_share = ceil_div(ceil_div(a.inner, stage), p.down.splits);
    const bool pack = !begin_at(a.x, a.x_stride, a.tokens, b, 8);
    p.x = pack ? packed : const_cast<void*>(a.x);
    p.x_stride = pack ? size.x_stride : a.x_stride;
    static_assert(kMaxPairs <= 2 * 1024 && FMB_MAX_GROUPS <= 1024, "a thread for every expert and every two pairs");
    const int list_threads = (int)up_to(std::max({a.experts, (a.tokens * a.top + 1) / 2, pack ? 256 : 1}), 32);
    FMB_CUDA_CHECK(launch_early(k_list_pairs<T>, pack ? a.tokens + 1 : 1, list_threads, 0, stream, p, (int)size.control, packed));
    FMB_LAUNCH_CHECK();
    // whole pieces of 16 bytes, at multiples of 16
    auto pieces = [&](const void* base, long long row, long long group, int rows, int columns) {
        return columns * b % 16 == 0 && begin_at(base, row, rows, b, 16) && begin_at(base, group, a.experts, b, 16);
    };
    const bool wide = pieces(a.w_up, a.up_row_stride, a.up_group_stride, a.width, a.inner) && pieces(a.w_down, a.down_row_stride, a.down_group_stride, a.inner, a.width);
    const long long most = std::min<long long>(a.experts, (long long)a.tokens * a.top) * (p.up.blocks * p.up.splits + p.down.blocks * p.down.splits);
    const int grid = (int)std::min<long long>(most, 2 * grp::sm_count());
    const auto kernel = wide ? k_experts<T, true> : k_experts<T, false>;
    const int smem = wide ? sizeof(Smem<T, true>) : sizeof(Smem<T, false>);
    FMB_CUDA_CHECK(opt_in_shared_memory((const void*)kernel, smem));
    FMB_CUDA_CHECK(launch_early(kernel, grid, kThreads, smem, stream, p));
    FMB_LAUNCH_CHECK();
    return FMB_OK;
}

bool fits(const void* base, long long stride, int bytes) { return ((uintptr_t)base & 15) == 0 && stride * bytes % 16 == 0; }

template <typename T, int TOKENS>
int route(const fmb_route_t& a, cudaStream_t stream) {
    int rows = 1;
    while (2 * rows * ((a.experts + 7) / 8) <= kThreads) rows *= 2;
    const int smem = TOKENS * std::max(kRouteChunk, rows * ((a.experts + 7) / 8) * 8) * (int)sizeof(float);
    FMB_CUDA_CHECK(opt_in_shared_memory((const void*)k_route<T, TOKENS>, TOKENS * kThreads * 8 * (int)sizeof(float)));
    cudaLaunchConfig_t config = {};
    cudaLaunchAttribute cluster;
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = kMaxCluster;
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    config.gridDim = dim3((unsigned)ceil_div(a.tokens, TOKENS) * kMaxCluster);
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    config.attrs = &cluster;
    config.numAttrs = 1;
    FMB_CUDA_CHECK(cudaLaunchKernelEx(&config, k_route<T, TOKENS>, a, (int)fits(a.router, a.router_stride, sizeof(T)), rows));
    FMB_LAUNCH_CHECK();
    return FMB_OK;
}

template <typename T, int MT, int COLUMNS, int KEYS>
int route_many(const fmb_route_t& a, cudaStream_t stream) {
    const auto kernel = k_route_many<T, MT, COLUMNS, KEYS>;
    constexpr int kRing = kRouteRing<MT, COLUMNS>, kLogits = 16 * MT * route_row(32 * KEYS) * (int)sizeof(float);
    constexpr int kSmem = KEYS * 32 <= COLUMNS ? std::max(kRing, kLogits) : kRing + kLogits;
    static_assert(kSmem <= 227 * 1024, "shared memory of a CTA");
    FMB_CUDA_CHECK(opt_in_shared_memory((const void*)kernel, kSmem));
    const int blocks = ceil_div(a.tokens, 16 * MT), stages = ceil_div(a.width, kRouteDepth<T>);
    // CTAs that share the depth, while there are SMs for them, for two each where they fit (8,192 tokens of 2,048, 64 experts: 18.9 us, and 20.6 with
    // one each)
    constexpr int kResident = std::min(2, 227 * 1024 / kSmem);
    int share = 1;
    while (share < kMaxCluster && 2 * share * blocks <= kResident * grp::sm_count() && 2 * share <= stages) share *= 2;
    cudaLaunchConfig_t config = {};
    cudaLaunchAttribute cluster;
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = share;
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    config.gridDim = dim3((unsigned)(blocks * share));
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = kSmem;
    config.stream = stream;
    config.attrs = &cluster;
    config.numAttrs = share > 1;
    FMB_CUDA_CHECK(cudaLaunchKernelEx(&config, kernel, a, (int)fits(a.x, a.x_stride, sizeof(T)), (int)fits(a.router, a.router_stride, sizeof(T)), share));
    FMB_LAUNCH_CHECK();
    return FMB_OK;
}

template <typename T>
int route(const fmb_route_t& a, cudaStream_t stream) {
    // us by blocks of many tokens, and by clusters for a few, bf16: 64 tokens and 64 experts of 2,048 8.7, 7.1; 64 and 128 of 4,096 13.7, 12.2; 8 and 256 20,
    // 13; 64 and 256 21, 24; 128 and 256 21, 34; 4 and 1,024 of 2,048 28, 51 (rows at whole pieces of 16 bytes; 1 and 300 of 4,096, which are not, 66 by
    // blocks). fp32: 128 and 256 of 4,096 72, 37; 1,024 and 64 of 2,048 23, 45
    const bool pieces = fits(a.x, a.x_stride, sizeof(T)) && fits(a.router, a.router_stride, sizeof(T));
    if (a.tokens > 128 || (sizeof(T) == 2 && pieces && (a.tokens * a.experts > 8192 || a.experts > 256)))
        return a.experts <= 64    ? route_many<T, 4, 64, 2>(a, stream)
               : a.experts <= 128 ? route_many<T, 4, 128, 4>(a, stream)
               : a.experts <= 256 ? route_many<T, 4, 256, 8>(a, stream)
                                  : route_many<T, 2, 128, 32>(a, stream);
    // by what the tokens would read of R one by one (us with one, two, four, eight tokens a cluster: 64 tokens and 32 experts of 4,096: 7.7, -, 10.9, -;
    // 64 and 256: -, -, 24, -; 128 and 256: 56, -, -, 35)
    const int logits = a.tokens * a.experts;
    return logits <= 4096 ? route<T, 1>(a, stream) : logits <= 8192 ? route<T, 2>(a, stream)
           : logits <= 16384 ? route<T, 4>(a, stream) : route<T, 8>(a, stream);
}

}  // namespace
}  // namespace exp_layer
}  // namespace fmb

using namespace fmb;
using namespace fmb::exp_layer;

extern "C" FMB_API int fmb_route_rows(const fmb_route_t* a, fmb_stream_t stream) {
    FMB_REQUIRE(a, "fmb_route_rows: null argument");
    FMB_REQUIRE(a->type >= FMB_TYPE_F32 && a->type <= FMB_TYPE_F16, "fmb_route_rows: type");
    FMB_REQUIRE(a->tokens >= 0 && a->tokens <= (1 << 24), "fmb_route_rows: more than 2^24 tokens");
    FMB_REQUIRE(a->width >= 1 && a->width <= (1 << 20), "fmb_route_rows: 1 to 2^20 columns");
    FMB_REQUIRE(a->experts >= 1 && a->experts <= FMB_MAX_GROUPS, "fmb_route_rows: 1 to FMB_MAX_GROUPS experts");
    FMB_REQUIRE(a->top >= 1 && a->top <= FMB_MAX_TOP && a->top <= a->experts, "fmb_route_rows: 1 to FMB_MAX_TOP choices, of the experts there are");
    if (a->tokens == 0) return FMB_OK;
    FMB_REQUIRE(a->x && a->router && a->chosen && a->weights, "fmb_route_rows: null argument");
    FMB_REQUIRE((a->tokens == 1 || a->x_stride >= a->width) && (a->width == 1 || a->router_stride >= a->experts), "fmb_route_rows: rows overlap");
    return a->type == FMB_TYPE_F32    ? route<float>(*a, (cudaStream_t)stream)
           : a->type == FMB_TYPE_BF16 ? route<__nv_bfloat16>(*a, (cudaStream_t)stream)
                                      : route<__half>(*a, (cudaStream_t)stream);
}

namespace {

int check_layer(const fmb_experts_t* a) {
    FMB_REQUIRE(a, "fmb_expert_layer: null argument");
    FMB_REQUIRE(a->type >= FMB_TYPE_F32 && a->type <= FMB_TYPE_F16, "fmb_expert_layer: type");
    FMB_REQUIRE(a->tokens >= 0 && a->tokens <= FMB_MAX_LAYER_TOKENS, "fmb_expert_layer: more than FMB_MAX_LAYER_TOKENS tokens");
    FMB_REQUIRE(a->width >= 1 && a->width <= (1 << 17) && a->inner >= 1 && a->inner <= (1 << 17), "fmb_expert_layer: 1 to 2^17 columns");
    FMB_REQUIRE(a->experts >= 1 && a->experts <= FMB_MAX_GROUPS, "fmb_expert_layer: 1 to FMB_MAX_GROUPS experts");
    FMB_REQUIRE(a->top >= 1 && a->top <= FMB_MAX_TOP, "fmb_expert_layer: 1 to FMB_MAX_TOP choices");
    return FMB_OK;
}

}  // namespace

extern "C" FMB_API long long fmb_expert_layer_scratch(const fmb_experts_t* a) {
    if (check_layer(a) || a->tokens == 0) return 0;
    const Sizes s = sizes_of(*a);
    return s.control + s.lists + s.h + s.parts + s.up_parts + s.x;
}

extern "C" FMB_API int fmb_expert_layer(const fmb_experts_t* a, fmb_stream_t stream) {
    const int rc = check_layer(a);
    if (rc || a->tokens == 0) return rc;
    FMB_REQUIRE(a->x && a->w_up && a->w_down && a->chosen && a->weights && a->y && a->scratch, "fmb_expert_layer: null argument");
    FMB_REQUIRE(a->tokens == 1 || (a->x_stride >= a->width && a->y_stride >= a->width), "fmb_expert_layer: rows overlap");
    const long long far = (1ll << 31) / 4 - 1;
    FMB_REQUIRE(a->up_row_stride >= 0 && a->up_row_stride <= far && a->down_row_stride >= 0 && a->down_row_stride <= far, "fmb_expert_layer: rows of weights more than 2^29 apart");
    FMB_REQUIRE(((uintptr_t)a->scratch & 15) == 0, "fmb_expert_layer: scratch starts at a multiple of 16 bytes");
    return a->type == FMB_TYPE_F32    ? layer<float>(*a, (cudaStream_t)stream)
           : a->type == FMB_TYPE_BF16 ? layer<__nv_bfloat16>(*a, (cudaStream_t)stream)
                                      : layer<__half>(*a, (cudaStream_t)stream);
}
