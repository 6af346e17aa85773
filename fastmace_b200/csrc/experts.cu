// An expert layer for a few tokens: routing, and the experts' two matrices with the gate between them.
//
//   route:   l = x R; the `top` largest of each token, ties to the lowest number; weights softmax(l) of the chosen, or of all
//   layer:   y[t] = sum_j w[t, j] (silu(x Wg) * (x Wu)) Wd of expert e(t, j)
//
// What bounds the layer is the weights of the experts that are chosen, read once from memory. One launch does both products:
// units of 32 gate columns with the 32 columns they multiply, then units of 64 columns of the second matrix, handed out in that order by
// a counter. A unit of the second kind waits for the first ones of its expert only; those were handed out before it, so they
// are done or under way and the wait ends, however few CTAs run at a time.
//
// A unit is [64 columns] x [8 or 16 rows] over the whole depth, which the eight warps of a CTA share. Weights go from memory to the
// registers that the tensor core reads them from: a lane loads eight neighbouring columns of as many rows of the matrix as a step has for
// it, and two permutes make pairs along the depth of them. Columns of the matrix are the MMA's rows, tokens its columns, of which it
// has eight: mma.sync suits that shape (tcgen05 would take 128 columns from shared memory for the same bytes).
//
// Numbers: 16-bit products are exact in fp32. What passes between the products, h, is not rounded to the type of the weights: it is a pair of
// bfloat16 (17 bits, any float32's range) against bfloat16 weights, a pair of tf32 against float16 ones, which are exact in tf32.
// float32 operands are pairs of tf32 (22 bits), of whose four products the smallest is left out.

#include "grouped.cuh"

#include <algorithm>
#include <type_traits>

namespace fmb {
namespace exp_layer {

namespace {

constexpr int kThreads = 256, kWarps = 8;
constexpr int kUnit = 64;                        // columns of a unit
constexpr long long kSpins = 1ll << 22;          // polls of a wait, each of 32 ns or more, before a CTA gives up

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T rounded(float x) { return grp::from_float<T>(x); }
template <> __device__ __forceinline__ float rounded<float>(float x) { return x; }
template <typename T> __device__ __forceinline__ T zero() { return T(0.0f); }

// --------------------------------------------------------------------------------------------------------------- route

constexpr int kCluster = 8;                      // CTAs that share the depth of a token's logits

// eight values from `at` on, of which `live` exist
template <typename T>
__device__ __forceinline__ void load_eight(const T* __restrict__ at, int live, bool wide, float (&v)[8]) {
    if (wide && live >= 8) {
        uint4 in[sizeof(T) / 2];
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) in[i] = __ldg(reinterpret_cast<const uint4*>(at) + i);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_float(reinterpret_cast<const T*>(in)[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < live ? to_float(at[i]) : 0.0f;
    }
}

// floats in an order of unsigned numbers; NaN below all
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t bits = __float_as_uint(x + 0.0f);              // (-0 and 0 are equal)
    return x != x ? 0u : bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

// A cluster per token: each CTA takes an eighth of the depth, threads by packs of eight experts and rows of R.
template <typename T>
__global__ void __launch_bounds__(kThreads)
k_route(fmb_route_t a, int wide, int rows) {
    __shared__ float sums[kThreads * 8];
    __shared__ float logits[FMB_MAX_GROUPS];
    const int token = blockIdx.x / kCluster, rank = blockIdx.x % kCluster, packs = (a.experts + 7) / 8;
    const int pack = threadIdx.x % packs, row = threadIdx.x / packs;
    const T* const x = (const T*)a.x + token * a.x_stride;
    const int begin = (int)((long long)a.width * rank / kCluster), end = (int)((long long)a.width * (rank + 1) / kCluster);
    float sum[8] = {};
    if (row < rows) {
        for (int k0 = begin + row; k0 < end; k0 += 4 * rows) {
            float w[4][8], v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = k0 + j * rows;
                v[j] = k < end ? to_float(x[k]) : 0.0f;
                load_eight((const T*)a.router + k * a.router_stride + 8 * pack, k < end ? a.experts - 8 * pack : 0, wide, w[j]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (k0 + j * rows < end) sum[i] = fmaf(v[j], w[j][i], sum[i]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) sums[row * packs * 8 + 8 * pack + i] = sum[i];
    }
    for (int half = rows / 2; half > 0; half /= 2) {
        __syncthreads();
        for (int i = threadIdx.x; i < half * packs * 8; i += kThreads) sums[i] += sums[i + half * packs * 8];
    }
    // the CTAs' sums, in their order, by the first
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank == 0) {
        const uint32_t here = (uint32_t)__cvta_generic_to_shared(sums);
        for (int e = threadIdx.x; e < a.experts; e += kThreads) {
            float part[kCluster];
#pragma unroll
            for (int c = 0; c < kCluster; ++c) {
                uint32_t there;
                asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(here + 4 * e), "r"(c));
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(part[c]) : "r"(there) : "memory");
            }
            float all = part[0];
#pragma unroll
            for (int c = 1; c < kCluster; ++c) all += part[c];
            logits[e] = all;
        }
    }
    // (their shared memory lives until it has been read)
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank != 0 || threadIdx.x >= 32) return;
    const int lane = threadIdx.x;
    unsigned taken = 0;                          // of this lane's experts lane, lane + 32, ...
    float first = 0.0f, total = 0.0f, mine = 0.0f;
    int chosen = 0;
    for (int j = 0; j < a.top; ++j) {
        unsigned long long best = 0;             // logit, then the lowest number
        for (int i = 0; i * 32 + lane < a.experts; ++i)
            if (!(taken >> i & 1)) best = max(best, (unsigned long long)ordered(logits[i * 32 + lane]) << 32 | (0xffffffffu - (i * 32 + lane)));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        const int e = (int)(0xffffffffu - (uint32_t)best);
        if ((e & 31) == lane) taken |= 1u << (e >> 5);
        const float l = logits[e];
        if (j == 0) first = l;
        const float p = expf(l - first);
        if (a.normalise) total += p;
        if (lane == j) {
            chosen = e;
            mine = p;
        }
    }
    if (!a.normalise) {
        for (int e = lane; e < a.experts; e += 32) total += expf(logits[e] - first);
        total = warp_sum(total);
    }
    if (lane < a.top) {
        a.chosen[token * (long long)a.top + lane] = chosen;
        a.weights[token * (long long)a.top + lane] = mine / total;
    }
}

// --------------------------------------------------------------------------------------------------------------- layer

__device__ __forceinline__ void mma_16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// x = hi + lo + less than 2^-22 |x|; an infinity or NaN stays in hi alone
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
    const float rest = fabsf(x) <= 3.4e38f ? x - __uint_as_float(hi) : 0.0f;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(rest));
}

// What a lane brings of a step: kRows neighbouring rows of the matrix, eight columns of each. A step has 4 kRows rows.
template <typename T> struct Step { static constexpr int kRows = sizeof(T) == 4 ? 4 : 8, kDepth = 4 * kRows, kWords = sizeof(T) == 4 ? 8 : 4; };

template <typename T, bool WIDE>
__device__ __forceinline__ void load_weights(const T* __restrict__ w, long long stride, int k, int depth, int live, uint32_t (&v)[Step<T>::kRows][Step<T>::kWords]) {
#pragma unroll
    for (int j = 0; j < Step<T>::kRows; ++j) {
        const T* const at = w + (long long)j * stride;
        const int here = k + j < depth ? live : 0;
        if (WIDE) {
            // (rows and columns by whole packs)
#pragma unroll
            for (int i = 0; i < Step<T>::kWords; i += 4) {
                uint4 in = make_uint4(0, 0, 0, 0);
                if (here > 0) asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                                           : "=r"(in.x), "=r"(in.y), "=r"(in.z), "=r"(in.w) : "l"(reinterpret_cast<const uint4*>(at) + i / 4));
                v[j][i] = in.x; v[j][i + 1] = in.y; v[j][i + 2] = in.z; v[j][i + 3] = in.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < Step<T>::kWords; ++i) {
                if constexpr (sizeof(T) == 4) {
                    v[j][i] = i < here ? __float_as_uint(__ldg((const float*)at + i)) : 0u;
                } else {
                    const uint32_t low = 2 * i < here ? __ldg((const uint16_t*)at + 2 * i) : 0u, high = 2 * i + 1 < here ? __ldg((const uint16_t*)at + 2 * i + 1) : 0u;
                    v[j][i] = low | high << 16;
                }
            }
        }
    }
}

// A unit's rows for a step, of which a lane has Step::kRows of the depth, of one row per eight. Rows of x:
template <typename T> struct RowsOfX {
    static constexpr int kRegs = 4;
    uint32_t v[kRegs];

    __device__ __forceinline__ void load(const T* __restrict__ row, int k, int depth, bool wide) {
        constexpr int kRows = Step<T>::kRows;
        const int live = row ? depth - k : 0;
        if (wide && live >= kRows) {
            const uint4 in = __ldg(reinterpret_cast<const uint4*>(row + k));
            v[0] = in.x; v[1] = in.y; v[2] = in.z; v[3] = in.w;
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = i < live ? __float_as_uint(__ldg((const float*)row + k + i)) : 0u;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t low = 2 * i < live ? __ldg((const uint16_t*)row + k + 2 * i) : 0u;
                const uint32_t high = 2 * i + 1 < live ? __ldg((const uint16_t*)row + k + 2 * i + 1) : 0u;
                v[i] = low | high << 16;
            }
        }
    }
};

// rows of h, which the other CTAs of this launch have written (so never by way of L1): for bfloat16 weights two bfloat16 a value, of
// which the upper halves of eight values lie before their lower ones; else float32
template <typename T> struct RowsOfH {
    static constexpr int kRegs = Step<T>::kRows;
    uint32_t v[kRegs];

    __device__ __forceinline__ void load(const float* __restrict__ row, int k, int, bool) {
#pragma unroll
        for (int i = 0; i < kRegs; i += 4) {
            const uint4 in = row ? __ldcg(reinterpret_cast<const uint4*>(row + k + i)) : make_uint4(0, 0, 0, 0);
            v[i] = in.x; v[i + 1] = in.y; v[i + 2] = in.z; v[i + 3] = in.w;
        }
    }
};

// acc[i][n]: columns 2 i and 2 i + 1 of the lanes' eight, rows of block n
template <typename T, int NB>
__device__ __forceinline__ void multiply_x(float (&acc)[4][NB][4], const uint32_t (&w)[Step<T>::kRows][Step<T>::kWords], const RowsOfX<T> (&x)[NB]) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t a[4] = {__byte_perm(w[4 * s][i], w[4 * s + 1][i], 0x5410), __byte_perm(w[4 * s][i], w[4 * s + 1][i], 0x7632),
                                       __byte_perm(w[4 * s + 2][i], w[4 * s + 3][i], 0x5410), __byte_perm(w[4 * s + 2][i], w[4 * s + 3][i], 0x7632)};
#pragma unroll
                for (int n = 0; n < NB; ++n) mma_16(acc[i][n], a, x[n].v[2 * s], x[n].v[2 * s + 1], T());
            }
    } else {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            uint32_t b[NB][2][2];
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int q = 0; q < 2; ++q) split_tf32(__uint_as_float(x[n].v[2 * s + q]), b[n][0][q], b[n][1][q]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) split_tf32(__uint_as_float(w[2 * s + q / 2][2 * i + q % 2]), hi[q], lo[q]);
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    mma_tf32(acc[i][n], hi, b[n][1][0], b[n][1][1]);
                    mma_tf32(acc[i][n], lo, b[n][0][0], b[n][0][1]);
                    mma_tf32(acc[i][n], hi, b[n][0][0], b[n][0][1]);
                }
            }
        }
    }
}

template <typename T, int NB>
__device__ __forceinline__ void multiply_h(float (&acc)[4][NB][4], const uint32_t (&w)[Step<T>::kRows][Step<T>::kWords], const RowsOfH<T> (&h)[NB]) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t a[4] = {__byte_perm(w[4 * s][i], w[4 * s + 1][i], 0x5410), __byte_perm(w[4 * s][i], w[4 * s + 1][i], 0x7632),
                                       __byte_perm(w[4 * s + 2][i], w[4 * s + 3][i], 0x5410), __byte_perm(w[4 * s + 2][i], w[4 * s + 3][i], 0x7632)};
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    mma_16(acc[i][n], a, h[n].v[4 + 2 * s], h[n].v[4 + 2 * s + 1], T());
                    mma_16(acc[i][n], a, h[n].v[2 * s], h[n].v[2 * s + 1], T());
                }
            }
    } else if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            uint32_t b[NB][2][2];
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int q = 0; q < 2; ++q) split_tf32(__uint_as_float(h[n].v[2 * s + q]), b[n][0][q], b[n][1][q]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t a[4];
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const float2 two = __half22float2(*reinterpret_cast<const __half2*>(&w[2 * s + q][i]));
                    a[2 * q] = __float_as_uint(two.x);
                    a[2 * q + 1] = __float_as_uint(two.y);
                }
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    mma_tf32(acc[i][n], a, b[n][1][0], b[n][1][1]);
                    mma_tf32(acc[i][n], a, b[n][0][0], b[n][0][1]);
                }
            }
        }
    } else {
        RowsOfX<T> x[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[n].v[i] = h[n].v[i];
        multiply_x<T, NB>(acc, w, x);
    }
}

struct Layer {
    fmb_experts_t a;
    int up_wide, down_wide, x_wide;
    int up_units, down_units;                    // of an expert
    long long h_stride, part_stride;             // floats of a row: the inner width, or the width, filled up to whole units
    int32_t* control;                            // next unit, CTAs that gave up; units of each expert that are done; experts of each column unit
    float* h;                                    // [tokens * top]
    float* parts;
};

// rows a reduction keeps of a column: chosen so that the lanes' stores fall on different banks
template <int NB> struct Turn { static constexpr int kStride = NB == 1 ? 8 : 24; };

// The sums over the depth of 64 columns and 8 NB rows, left in turn[column][row] by all warps: columns 8 g + j at place 8 j + g.
template <typename T, bool WIDE, int NB, bool UP>
__device__ __forceinline__ void product(const Layer& p, const T* __restrict__ w, long long stride, int live, int depth, const void* const (&rows)[NB], float* turn) {
    constexpr int kRows = Step<T>::kRows, kDepth = Step<T>::kDepth;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane & 3;
    using Rows = typename std::conditional<UP, RowsOfX<T>, RowsOfH<T>>::type;
    using From = typename std::conditional<UP, T, float>::type;
    float acc[4][NB][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[i][n][q] = 0.0f;
    uint32_t v[2][kRows][Step<T>::kWords];
    Rows x[2][NB];
    const int steps = (depth + kDepth - 1) / kDepth;
    auto bring = [&](int step, int slot) {
        const int k = step * kDepth + kRows * quad;
        load_weights<T, WIDE>(w + k * stride, stride, k, step < steps ? depth : 0, live, v[slot]);
#pragma unroll
        for (int n = 0; n < NB; ++n) x[slot][n].load(step < steps ? (const From*)rows[n] : nullptr, k, depth, p.x_wide);
    };
    bring(warp, 0);
#pragma unroll 2
    for (int step = warp, slot = 0; step < steps; step += kWarps, slot ^= 1) {
        bring(step + kWarps, slot ^ 1);
        if constexpr (UP) multiply_x<T, NB>(acc, v[slot], x[slot]);
        else multiply_h<T, NB>(acc, v[slot], x[slot]);
    }
    float* const mine = turn + warp * kUnit * Turn<NB>::kStride;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int b = 0; b < 2; ++b)
                *reinterpret_cast<float2*>(mine + ((2 * i + b) * 8 + (lane >> 2)) * Turn<NB>::kStride + 8 * n + 2 * quad) =
                    make_float2(acc[i][n][2 * b], acc[i][n][2 * b + 1]);
}

template <int NB>
__device__ __forceinline__ float sum_of(const float* turn, int place, int row) {
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sum += turn[(w * kUnit + place) * Turn<NB>::kStride + row];
    return sum;
}

constexpr int kMaxPairs = FMB_MAX_LAYER_TOKENS * FMB_MAX_TOP;
constexpr int kTurnFloats = kWarps * kUnit * 24;

template <typename T>
struct Smem {
    float turn[kTurnFloats];
    int pair[kMaxPairs];                         // pairs of token and choice, by expert
    int start[FMB_MAX_GROUPS + 1];
    int active[FMB_MAX_GROUPS];                  // experts that have pairs
    int warp_total[2][kWarps];
    int ticket[2], actives, flag;
};

// Which pairs belong to which expert, and which experts have any. Pairs of one expert stand in any order: their results do not
// depend on it.
template <typename T>
__device__ __forceinline__ void list_pairs(const Layer& p, Smem<T>& s) {
    const int experts = p.a.experts, pairs = p.a.tokens * p.a.top, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int e = threadIdx.x; e <= experts; e += kThreads) s.start[e] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < pairs; i += kThreads) {
        const int e = __ldg(p.a.chosen + i);
        if (e >= 0 && e < experts) atomicAdd(s.start + e, 1);
    }
    __syncthreads();
    const int per = (experts + kThreads - 1) / kThreads, from = min(experts, (int)threadIdx.x * per), to = min(experts, from + per);
    int sum = 0, some = 0;
    for (int e = from; e < to; ++e) {
        sum += s.start[e];
        some += s.start[e] > 0;
    }
    int sums = sum, somes = some;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, sums, o), b = __shfl_up_sync(0xffffffffu, somes, o);
        if (lane >= o) sums += a, somes += b;
    }
    if (lane == 31) s.warp_total[0][warp] = sums, s.warp_total[1][warp] = somes;
    __syncthreads();
    int before = sums - sum, number = somes - some;
    for (int w = 0; w < warp; ++w) before += s.warp_total[0][w], number += s.warp_total[1][w];
    for (int e = from; e < to; ++e) {
        const int count = s.start[e];
        if (count > 0) s.active[number++] = e;
        before += count;
        s.start[e] = before;                     // the end: places are taken from there downwards
    }
    if (threadIdx.x == kThreads - 1) {
        s.start[experts] = before;
        s.actives = number;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < pairs; i += kThreads) {
        const int e = __ldg(p.a.chosen + i);
        if (e >= 0 && e < experts) s.pair[atomicSub(s.start + e, 1) - 1] = i;
    }
    __syncthreads();
}

__device__ __forceinline__ int load_acquire(const int32_t* at) {
    int v;
    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(at) : "memory");
    return v;
}

// 32 gate columns and those they multiply, for `count` (up to 8 NB) pairs from `first` on
template <typename T, bool WIDE, int NB>
__device__ __forceinline__ void up_unit(const Layer& p, Smem<T>& s, int expert, int block, int first, int count) {
    const fmb_experts_t& a = p.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c0 = 32 * block + 8 * (g & 3);
    const void* rows[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) rows[n] = 8 * n + g < count ? (const T*)a.x + (s.pair[first + 8 * n + g] / a.top) * a.x_stride : nullptr;
    const T* const w = (const T*)a.w_up + expert * a.up_group_stride + (g < 4 ? 0 : a.inner) + c0;
    product<T, WIDE, NB, true>(p, w, a.up_row_stride, a.inner - c0, a.width, rows, s.turn);
    __syncthreads();
    // warp j: columns j, 8 + j, 16 + j, 24 + j of the 32; a lane has one of them and one row of each eight
    const int column = 32 * block + 8 * (lane >> 3) + warp;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        const int row = 8 * n + (lane & 7);
        const float gate = sum_of<NB>(s.turn, 8 * warp + (lane >> 3), row), up = sum_of<NB>(s.turn, 8 * warp + 4 + (lane >> 3), row);
        if (row >= count) continue;
        const float h = column < a.inner ? gate / (1.0f + expf(-gate)) * up : 0.0f;
        float* const to = p.h + s.pair[first + row] * p.h_stride;
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            const __nv_bfloat16 hi = __float2bfloat16_rn(h);
            const float rest = fabsf(h) <= 3.3e38f ? h - __bfloat162float(hi) : 0.0f;
            __nv_bfloat16* const eight = (__nv_bfloat16*)(to + (column & ~7));
            eight[column & 7] = hi;
            eight[8 + (column & 7)] = __float2bfloat16_rn(rest);
        } else {
            to[column] = h;
        }
    }
}

template <typename T, bool WIDE, int NB>
__device__ __forceinline__ void down_unit(const Layer& p, Smem<T>& s, int expert, int block, int first, int count) {
    const fmb_experts_t& a = p.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c0 = kUnit * block + 8 * g;
    const void* rows[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) rows[n] = 8 * n + g < count ? p.h + s.pair[first + 8 * n + g] * p.h_stride : nullptr;
    product<T, WIDE, NB, false>(p, (const T*)a.w_down + expert * a.down_group_stride + c0, a.down_row_stride, a.width - c0, a.inner, rows, s.turn);
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int row = 8 * n + (lane & 7), at = 4 * q + (lane >> 3);
            const float sum = sum_of<NB>(s.turn, 8 * warp + at, row);
            if (row < count) p.parts[s.pair[first + row] * p.part_stride + kUnit * block + 8 * at + warp] = sum;
        }
}

// y of 64 columns: what the experts of each token have given, in the order of its choices
template <typename T>
__device__ __forceinline__ void combine(const Layer& p, int block) {
    const fmb_experts_t& a = p.a;
    const int c = kUnit * block + (threadIdx.x & (kUnit - 1));
    if (c >= a.width) return;
    for (int t = threadIdx.x / kUnit; t < a.tokens; t += kThreads / kUnit) {
        float sum = 0.0f;
        for (int j0 = 0; j0 < a.top; j0 += 4) {
            float v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int pair = t * a.top + j0 + j, e = j0 + j < a.top ? __ldg(a.chosen + pair) : -1;
                v[j] = e >= 0 && e < a.experts ? __ldg(a.weights + pair) * __ldcg(p.parts + pair * p.part_stride + c) : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) sum += v[j];
        }
        ((T*)a.y)[t * a.y_stride + c] = rounded<T>(sum);
    }
}

template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads, 2)
k_experts(const __grid_constant__ Layer p) {
    extern __shared__ __align__(16) uint8_t smem[];
    Smem<T>& s = *reinterpret_cast<Smem<T>*>(smem);
    const fmb_experts_t& a = p.a;
    int32_t* const next = p.control;
    int32_t* const done = p.control + 2;
    int32_t* const columns = done + a.experts;
    if (threadIdx.x == 0) s.ticket[0] = atomicAdd(next, 1);
    list_pairs(p, s);
    const int actives = s.actives, ups = actives * p.up_units, units = ups + actives * p.down_units;
    if (actives == 0) {                          // no expert is one
        for (long long i = blockIdx.x * (long long)kThreads + threadIdx.x; i < (long long)a.tokens * a.width; i += (long long)gridDim.x * kThreads)
            ((T*)a.y)[i / a.width * a.y_stride + i % a.width] = zero<T>();
        return;
    }
    for (int round = 0;; round ^= 1) {
        const int unit = s.ticket[round];
        if (unit >= units) return;
        const bool up = unit < ups;
        const int number = up ? unit / p.up_units : (unit - ups) / p.down_units;
        const int block = up ? unit % p.up_units : (unit - ups) % p.down_units;
        const int expert = s.active[number], first = s.start[expert];
        // (the starts have been counted down to where each expert's pairs begin)
        int end = s.start[a.experts];
        if (number + 1 < actives) end = s.start[s.active[number + 1]];
        if (threadIdx.x == 0) {
            s.ticket[round ^ 1] = atomicAdd(next, 1);
            int ready = 1;
            if (!up) {
                long long spins = 0;
                while (load_acquire(done + number) < p.up_units && ++spins < kSpins) __nanosleep(32);
                ready = spins < kSpins;
                if (!ready && a.status) atomicOr(a.status, (uint32_t)FMB_STATUS_TENSOR_TIMEOUT);
            }
            s.flag = ready;
        }
        __syncthreads();
        if (!s.flag) return;
        for (int at = first; at < end; at += 16) {
            const int count = min(16, end - at);
            if (at > first) __syncthreads();
            if (up) {
                if (count <= 8) up_unit<T, WIDE, 1>(p, s, expert, block, at, count);
                else up_unit<T, WIDE, 2>(p, s, expert, block, at, count);
            } else {
                if (count <= 8) down_unit<T, WIDE, 1>(p, s, expert, block, at, count);
                else down_unit<T, WIDE, 2>(p, s, expert, block, at, count);
            }
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            __threadfence();
            if (up) {
                atomicAdd(done + number, 1);
                s.flag = 0;
            } else {
                s.flag = atomicAdd(columns + block, 1) == actives - 1;
                __threadfence();
            }
        }
        __syncthreads();
        if (s.flag) combine<T>(p, block);
        __syncthreads();                         // the flag has been read
    }
}

long long up_to(long long n, long long step) { return (n + step - 1) / step * step; }

struct Sizes {
    long long control, h, parts;                 // in floats
    long long h_stride, part_stride;
};

Sizes sizes_of(const fmb_experts_t& a) {
    Sizes s;
    s.control = up_to(2 + a.experts + ceil_div(a.width, kUnit), 64);
    s.h_stride = up_to(a.inner, 32);
    s.part_stride = up_to(a.width, kUnit);
    s.h = up_to((long long)a.tokens * a.top * s.h_stride, 64);
    s.parts = (long long)a.tokens * a.top * s.part_stride;
    return s;
}

bool fits(const void* base, long long stride, int bytes) { return ((uintptr_t)base & 15) == 0 && stride * bytes % 16 == 0; }

template <typename T>
int layer(const fmb_experts_t& a, cudaStream_t stream) {
    const Sizes size = sizes_of(a);
    Layer p;
    p.a = a;
    p.control = (int32_t*)a.scratch;
    p.h = a.scratch + size.control;
    p.parts = p.h + size.h;
    p.h_stride = size.h_stride;
    p.part_stride = size.part_stride;
    p.up_units = ceil_div(a.inner, 32);
    p.down_units = ceil_div(a.width, kUnit);
    const int b = sizeof(T);
    p.x_wide = fits(a.x, a.tokens > 1 ? a.x_stride : 8, b);
    // whole packs of eight columns
    const bool wide = a.inner % 8 == 0 && a.width % 8 == 0 && fits(a.w_up, a.up_row_stride, b) && fits(a.w_down, a.down_row_stride, b) &&
                      (a.experts == 1 || (a.up_group_stride * b % 16 == 0 && a.down_group_stride * b % 16 == 0));
    FMB_CUDA_CHECK(cudaMemsetAsync(p.control, 0, size.control * 4, stream));
    const void* const kernel = wide ? (const void*)k_experts<T, true> : (const void*)k_experts<T, false>;
    FMB_CUDA_CHECK(opt_in_shared_memory(kernel, sizeof(Smem<T>)));
    const long long most = std::min<long long>(a.experts, (long long)a.tokens * a.top) * (p.up_units + p.down_units);
    const int grid = (int)std::min<long long>(most, 2 * grp::sm_count());
    if (wide) k_experts<T, true><<<grid, kThreads, sizeof(Smem<T>), stream>>>(p);
    else k_experts<T, false><<<grid, kThreads, sizeof(Smem<T>), stream>>>(p);
    FMB_LAUNCH_CHECK();
    return FMB_OK;
}

template <typename T>
int route(const fmb_route_t& a, cudaStream_t stream) {
    const int packs = (a.experts + 7) / 8;
    int rows = 1;
    while (2 * rows * packs <= kThreads) rows *= 2;
    cudaLaunchConfig_t config = {};
    cudaLaunchAttribute cluster;
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = kCluster;
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    config.gridDim = dim3((unsigned)a.tokens * kCluster);
    config.blockDim = dim3(kThreads);
    config.stream = stream;
    config.attrs = &cluster;
    config.numAttrs = 1;
    const int wide = fits(a.router, a.router_stride, sizeof(T));
    FMB_CUDA_CHECK(cudaLaunchKernelEx(&config, k_route<T>, a, wide, rows));
    FMB_LAUNCH_CHECK();
    return FMB_OK;
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
    return s.control + s.h + s.parts;
}

extern "C" FMB_API int fmb_expert_layer(const fmb_experts_t* a, fmb_stream_t stream) {
    const int rc = check_layer(a);
    if (rc || a->tokens == 0) return rc;
    FMB_REQUIRE(a->x && a->w_up && a->w_down && a->chosen && a->weights && a->y && a->scratch, "fmb_expert_layer: null argument");
    FMB_REQUIRE(a->tokens == 1 || (a->x_stride >= a->width && a->y_stride >= a->width), "fmb_expert_layer: rows overlap");
    FMB_REQUIRE(((uintptr_t)a->scratch & 15) == 0, "fmb_expert_layer: scratch starts at a multiple of 16 bytes");
    return a->type == FMB_TYPE_F32    ? layer<float>(*a, (cudaStream_t)stream)
           : a->type == FMB_TYPE_BF16 ? layer<__nv_bfloat16>(*a, (cudaStream_t)stream)
                                      : layer<__half>(*a, (cudaStream_t)stream);
}
