// nf_logprobs.cu -- nf_token_logprobs (include/nf_moe.h): log-probability of
// a given token, entropy and the greatest logits of every row.
#include "nf_kv.h"

#include "nf_common.cuh"
#include "nf_gemm_shared.cuh"
#include "nf_internal.h"

#include <cmath>

namespace nf {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTop = 32;

// A logit's place in the order of the top tokens: greater logits first, -0
// and +0 equal, a NaN behind everything; the lower index first among equals.
__device__ __forceinline__ uint32_t value_key(float x) {
    const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);
    return isnan(x) ? 0u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t order_key(float x, int64_t index) {
    return (static_cast<uint64_t>(value_key(x)) << 32) | (0xffffffffu - static_cast<uint32_t>(index));
}

template <bool BF16>
__device__ __forceinline__ float load_logit(const void* p, int64_t i) {
    return BF16 ? bf16_bits_to_f32(static_cast<const uint16_t*>(p)[i]) : static_cast<const float*>(p)[i];
}

template <typename T, typename F>
__device__ __forceinline__ T block_reduce(T v, T* s, F f) {
    for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    v = s[0];
    for (int w = 1; w < kThreads / 32; ++w) v = f(v, s[w]);
    return v;
}

// A cluster's share of a row: groups of 8 logits (16-byte vectors) dealt out to
// the cluster's threads in turn, and the row's ends, one logit a thread of the
// first CTA.
template <bool BF16>
struct Slice {
    const uint8_t* p;         // the row
    int64_t head, groups;     // logits before the first group, groups
    int64_t vocab, step;      // threads of the cluster
    __device__ __forceinline__ Slice(const void* row, int64_t n, int ranks) {
        constexpr int kSize = BF16 ? 2 : 4;
        p = static_cast<const uint8_t*>(row);
        vocab = n;
        head = min(n, static_cast<int64_t>((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / kSize);
        groups = (n - head) / 8;
        step = static_cast<int64_t>(ranks) * kThreads;
    }
    __device__ __forceinline__ int64_t index(int64_t g) const { return head + 8 * g; }
    __device__ __forceinline__ void load(int64_t g, uint4* w) const {
        const uint4* q = reinterpret_cast<const uint4*>(p + index(g) * (BF16 ? 2 : 4));
        w[0] = __ldg(q);
        if (!BF16) w[1] = __ldg(q + 1);
    }
    // the single logit at an end of thread t of the cluster, or -1
    __device__ __forceinline__ int64_t single(int64_t t) const {
        const int64_t i = t < head ? t : 8 * groups + t;
        return t < 32 && i < vocab ? i : -1;
    }
};
template <bool BF16>
__device__ __forceinline__ void unpack(const uint4* w, float* f) {
#pragma unroll
    for (int h = 0; h < (BF16 ? 1 : 2); ++h) {
        const uint32_t v[4] = {w[h].x, w[h].y, w[h].z, w[h].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (BF16) {
                f[2 * k] = __uint_as_float(v[k] << 16);
                f[2 * k + 1] = __uint_as_float(v[k] & 0xffff0000u);
            } else {
                f[4 * h + k] = __uint_as_float(v[k]);
            }
        }
    }
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFar = -1e28f;  // stands for any distance below: e^x is 0, and x times a sum of 2^31 is finite

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ float key_value(uint32_t k) {  // value_key's inverse; 0 is a NaN
    return k == 0 ? NAN : __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}

// Sums of a set of logits: m the greatest, s = sum e^(x - m), t = sum e^(x - m) (x - m).
struct Sums {
    float m, s, t;
};
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
    Sums r;
    r.m = fmaxf(a.m, b.m);
    const float mu = r.m == -INFINITY ? 0.f : r.m;
    const float da = fmaxf(a.m - mu, kFar), db = fmaxf(b.m - mu, kFar);
    const float fa = ex2(da * kLog2e), fb = ex2(db * kLog2e);
    r.s = a.s * fa + b.s * fb;
    r.t = (a.t + a.s * da) * fa + (b.t + b.s * db) * fb;
    return r;
}

// What a CTA tells the first one of its cluster.
struct Told {
    Sums sums;
    int count;
    uint64_t key[kMaxTop];
};

constexpr int kCandidates = 1024;

// Where `v` stands among n values of s, the greatest first (the values differ).
__device__ __forceinline__ int rank_of(uint64_t v, const uint64_t* s, int n) {
    int r = 0;
#pragma unroll 8
    for (int i = 0; i < n; ++i) r += s[i] > v;
    return r;
}

// One cluster per row, one pass over its logits.  A thread keeps the running
// maximum and sums of its logits; a NaN or +infinity makes its sums NaN by
// itself.  The top tokens need no second pass: the top-th greatest of the
// threads' maxima bounds them from below, and only the logits of the threads
// whose maximum reaches it (`top` of 256, but for equals) can be among them;
// the CTA looks at these once more.
// The floor is one read of the logits; what bounds it is the loads' latency and
// the top tokens behind them where all rows' CTAs run at the same time, the
// instructions issued (nine for two logits) with more rows, and a row's own
// latency with few.
// 256 rows of 151,552 F32 logits, top 5: 34.9 us, 4.45 TB/s; 4,001 rows of
// 32,003 BF16 logits: 63.5 us, 4.0 TB/s.  The CTAs an SM holds matter: F32 with
// 76 registers, so three, 48.2 us; BF16 with four 71.6, with five 66.4.
// Where a CTA's share holds fewer than `top` threads with a logit above
// -infinity, every logit is a candidate, and the CTA reads its share once more
// for every top token: with 1, 3 or 20 tokens left in each of the 256 rows, 384,
// 383 and 178 us at top 5 and 1,244 at top 20, against 37.
template <bool BF16>
__global__ void __launch_bounds__(kThreads, BF16 ? 6 : 4) token_logprobs_kernel(const void* __restrict__ logits,
                                                                  const uint32_t* __restrict__ epoch,
                                                                  int64_t epoch_bytes, int64_t stride,
                                                                  int64_t vocab, const int32_t* __restrict__ target,
                                                                  int top, float* __restrict__ logprob,
                                                                  float* __restrict__ entropy,
                                                                  int32_t* __restrict__ top_idx,
                                                                  float* __restrict__ top_lp) {
    __shared__ Told s_told;
    __shared__ __align__(16) uint32_t s_max[kThreads];
    __shared__ uint16_t s_hot[kThreads];
    __shared__ uint64_t s_cand[kCandidates];
    __shared__ uint64_t s_red[kThreads / 32];
    __shared__ float2 s_sums[kThreads / 32];
    __shared__ uint32_t s_wmax[kThreads / 32];
    __shared__ uint32_t s_bound;
    __shared__ int s_hots, s_count;
    uint32_t ranks;
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ranks));
    const int rank = static_cast<int>(cluster_ctarank());
    const int64_t row = blockIdx.x / ranks;
    const void* x = static_cast<const uint8_t*>(logits) + (epoch ? (*epoch & 1u) * epoch_bytes : 0) + row * stride * (BF16 ? 2 : 4);
    const Slice<BF16> part(x, vocab, ranks);
    const int64_t g0 = static_cast<int64_t>(rank) * kThreads;  // the CTA's first thread in the cluster
    const int64_t mine = g0 + threadIdx.x, single = part.single(mine);

    // ---- the thread's logits
    Sums u{-INFINITY, 0.f, 0.f};
    auto add = [&](float v, float mu) {
        const float d = v - mu, e = ex2(d * kLog2e);
        u.s += e;
        u.t = fmaf(e, fmaxf(d, kFar), u.t);
    };
    auto grow = [&](float m) {
        const float d = fmaxf(u.m - m, kFar), f = ex2(d * kLog2e);  // m = -infinity: d NaN becomes kFar, f 0
        u.t = (u.t + u.s * d) * f;
        u.s *= f;
        u.m = m;
    };
    // two logits at a time: the loop is bound by the instructions issued
    uint64_t s2 = 0, t2 = 0;
    const uint64_t l2 = f32x2_pack(kLog2e, kLog2e);
#pragma unroll 1
    for (int64_t g = mine; g < part.groups; g += 4 * part.step) {
        uint4 w[4][BF16 ? 1 : 2];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (g + k * part.step < part.groups) part.load(g + k * part.step, w[k]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (g + k * part.step >= part.groups) break;
            float f[8];
            unpack<BF16>(w[k], f);
            const float m = max3(max3(max3(u.m, f[0], f[1]), f[2], f[3]), max3(f[4], f[5], f[6]), f[7]);
            const float d = fmaxf(u.m - m, kFar), c = ex2(d * kLog2e);  // m = -infinity: d NaN becomes kFar, c 0
            const uint64_t c2 = f32x2_pack(c, c);
            t2 = mul_f32x2(fma_f32x2(s2, f32x2_pack(d, d), t2), c2);
            s2 = mul_f32x2(s2, c2);
            u.m = m;
            const float mu = m == -INFINITY ? 0.f : m;
            const uint64_t nm = f32x2_pack(-mu, -mu);
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const uint64_t x2 = add_f32x2(f32x2_pack(f[e], f[e + 1]), nm), y2 = mul_f32x2(x2, l2);
                const uint64_t e2 = f32x2_pack(ex2(f32x2_lo(y2)), ex2(f32x2_hi(y2)));
                s2 = add_f32x2(s2, e2);
                t2 = fma_f32x2(e2, f32x2_pack(fmaxf(f32x2_lo(x2), kFar), fmaxf(f32x2_hi(x2), kFar)), t2);
            }
        }
    }
    u.s = f32x2_lo(s2) + f32x2_hi(s2);
    u.t = f32x2_lo(t2) + f32x2_hi(t2);
    if (single >= 0) {
        const float f = load_logit<BF16>(x, single);
        grow(fmaxf(u.m, f));
        add(f, u.m == -INFINITY ? 0.f : u.m);
    }

    // ---- the CTA's sums
    const bool any = mine < part.groups || single >= 0;
    // 0: no logit; a NaN or -infinity alone is 1 at least
    const uint32_t best = any ? max(1u, value_key(u.m)) : 0u;
    const uint32_t warp_best = __reduce_max_sync(0xffffffffu, best);
    s_max[threadIdx.x] = best;
    if ((threadIdx.x & 31) == 0) s_wmax[threadIdx.x >> 5] = warp_best;
    if (threadIdx.x == 0) s_hots = s_count = 0;
    __syncthreads();
    uint32_t top_key = s_wmax[0];
#pragma unroll
    for (int w = 1; w < kThreads / 32; ++w) top_key = max(top_key, s_wmax[w]);
    grow(fmaxf(u.m, key_value(top_key)));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        u.s += __shfl_xor_sync(0xffffffffu, u.s, o);
        u.t += __shfl_xor_sync(0xffffffffu, u.t, o);
    }
    if ((threadIdx.x & 31) == 0) s_sums[threadIdx.x >> 5] = make_float2(u.s, u.t);

    // ---- the CTA's top tokens
    if (top > 0) {
        // the top-th greatest of the threads' maxima (0 if fewer have a logit), bit by bit, by the first warp
        if (threadIdx.x < 32) {
            uint32_t b = top_key;
            if (top > 1) {
                const uint4 k0 = *reinterpret_cast<const uint4*>(s_max + 8 * threadIdx.x);
                const uint4 k1 = *reinterpret_cast<const uint4*>(s_max + 8 * threadIdx.x + 4);
                b = 0;
#pragma unroll 1
                for (uint32_t bit = 0x80000000u; bit != 0; bit >>= 1) {
                    const uint32_t c = b | bit;
                    const uint32_t n = (k0.x >= c) + (k0.y >= c) + (k0.z >= c) + (k0.w >= c) + (k1.x >= c) + (k1.y >= c) +
                                       (k1.z >= c) + (k1.w >= c);
                    if (__reduce_add_sync(0xffffffffu, n) >= static_cast<uint32_t>(top)) b = c;
                }
            }
            if (threadIdx.x == 0) s_bound = b;
        }
        __syncthreads();
        uint32_t bound = s_bound;
        if (bound <= value_key(-INFINITY)) bound = 0;  // -infinities and NaNs among the top: look at all
        if (any && best >= bound) s_hot[atomicAdd(&s_hots, 1)] = static_cast<uint16_t>(threadIdx.x);
        __syncthreads();
        // calls f(logit, index) for the hot threads' logits, all threads of the CTA sharing them
        const int hots = s_hots;
        const int64_t per = (part.groups + part.step - 1) / part.step, work = hots * (per + 1);
        auto each = [&](auto&& f) {
#pragma unroll 1
            for (int64_t i0 = threadIdx.x; i0 < work; i0 += 2 * kThreads) {
                uint4 w[2][BF16 ? 1 : 2];
                int64_t at[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int64_t i = i0 + k * kThreads;
                    const int64_t j = i < work ? i / hots : per + 1, t = g0 + s_hot[i < work ? i - j * hots : 0];
                    const int64_t g = t + j * part.step;
                    at[k] = -1;
                    if (j < per && g < part.groups) {
                        at[k] = part.index(g);
                        part.load(g, w[k]);
                    }
                    const int64_t one = j == per ? part.single(t) : -1;
                    if (one >= 0) f(load_logit<BF16>(x, one), one);
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if (at[k] < 0) continue;
                    float y[8];
                    unpack<BF16>(w[k], y);
#pragma unroll
                    for (int e = 0; e < 8; ++e) f(y[e], at[k] + e);
                }
            }
        };
        each([&](float f, int64_t i) {
            if (value_key(f) >= bound) {
                const int c = atomicAdd(&s_count, 1);
                if (c < kCandidates) s_cand[c] = order_key(f, i);
            }
        });
        __syncthreads();
        const int count = s_count;
        if (count <= kCandidates) {
#pragma unroll 1
            for (int c = threadIdx.x; c < count; c += kThreads) {
                const uint64_t k = s_cand[c];
                const int r = rank_of(k, s_cand, count);
                if (r < top) s_told.key[r] = k;
            }
            if (threadIdx.x == 0) s_told.count = min(count, top);
        } else {
            // many equal logits: one token at a time
            uint64_t last = ~0ull;
#pragma unroll 1
            for (int r = 0; r < top; ++r) {
                uint64_t next = 0;
                each([&](float f, int64_t i) {
                    const uint64_t k = order_key(f, i);
                    if (k < last && k > next) next = k;
                });
                last = block_reduce(next, s_red, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
                if (threadIdx.x == 0) s_told.key[r] = last;
            }
            if (threadIdx.x == 0) s_told.count = top;
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kThreads / 32; ++w) {
            u.s += s_sums[w].x;
            u.t += s_sums[w].y;
        }
        s_told.sums = u;
    }
    // ---- the row's, in the first CTA
    if (ranks > 1) cluster_sync();
    else __syncthreads();
    if (rank == 0) {
        if (ranks > 1) {
            u = s_told.sums;
            int n = 0;
            for (uint32_t c = 0; c < ranks; ++c) {
                const uint32_t base = smem_in_cta(&s_told, c);
                Sums o;
                asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(o.m), "=f"(o.s) : "r"(base) : "memory");
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o.t) : "r"(base + 8) : "memory");
                if (c > 0) u = join(u, o);
                if (top > 0) {
                    int count;
                    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(count) : "r"(base + 12) : "memory");
                    if (static_cast<int>(threadIdx.x) < count) {
                        uint64_t k;
                        asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(k) : "r"(base + 16 + 8 * threadIdx.x) : "memory");
                        s_cand[n + threadIdx.x] = k;
                    }
                    n += count;
                }
            }
            __syncthreads();
            if (static_cast<int>(threadIdx.x) < n) {
                const uint64_t k = s_cand[threadIdx.x];
                const int r = rank_of(k, s_cand, n);
                if (r < top) s_told.key[r] = k;
            }
            __syncthreads();
        } else {
            u = s_told.sums;
        }
        const float ls = u.m == -INFINITY || isinf(u.m) ? NAN : logf(u.s);
        if (threadIdx.x == 0) {
            if (logprob) {
                const int32_t id = target[row];
                logprob[row] = id >= 0 && id < vocab ? (load_logit<BF16>(x, id) - u.m) - ls : NAN;
            }
            if (entropy) entropy[row] = ls - u.t / u.s;
        }
        if (static_cast<int>(threadIdx.x) < top) {
            const uint64_t k = s_told.key[threadIdx.x];
            const int32_t id = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(k));
            top_idx[row * top + threadIdx.x] = id;
            top_lp[row * top + threadIdx.x] = (load_logit<BF16>(x, id) - u.m) - ls;
        }
    }
    if (ranks > 1) cluster_sync();  // the others' shared memory has been read
}

}  // namespace

cudaError_t launch_token_logprobs(const void* logits, int type, int64_t stride, int rows, int64_t vocab,
                                  const int32_t* target, int top, float* logprob, float* entropy, int32_t* top_idx,
                                  float* top_lp, cudaStream_t st, const uint32_t* epoch, int64_t epoch_bytes) {
    if (rows <= 0) return cudaSuccess;
    // clusters give a few rows every SM: two CTAs on each, as long as each has 4,096 logits (256 rows of 151,552 logits:
    // 36.3 us with one CTA a row, 34.9 with two, 43.0 with four, 65.8 with eight)
    unsigned ranks = 1;
    while (ranks < 8 && static_cast<int64_t>(rows) * ranks < 2 * 148 && vocab / (2 * ranks) >= 4096) ranks *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(rows) * ranks);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, type == NF_DTYPE_BF16 ? token_logprobs_kernel<true> : token_logprobs_kernel<false>,
                              logits, epoch, epoch_bytes, stride, vocab, target, top, logprob, entropy, top_idx, top_lp);
}

}  // namespace nf

using namespace nf;

extern "C" {

int64_t nf_token_logprobs_workspace(int rows, int64_t vocab, int top) {
    return rows < 0 || vocab < 1 || top < 0 || top > kMaxTop ? 0 : 16;
}

int nf_token_logprobs(const void* logits, int logits_type, int64_t row_stride, int rows, int64_t vocab,
                      const int32_t* target, int top, float* logprob, float* entropy, int32_t* top_idx, float* top_lp,
                      void* work, int64_t work_bytes, void* stream) {
    kv_clear_error();
    if (logits_type != NF_DTYPE_F32 && logits_type != NF_DTYPE_BF16)
        return kv_fail(NF_ERR_INVALID, "unknown logits type %d", logits_type);
    if (rows < 0) return kv_fail(NF_ERR_INVALID, "rows must be >= 0");
    if (vocab < 1 || vocab > 0x7fffffffll) return kv_fail(NF_ERR_SHAPE, "vocab must be in [1, 2^31)");
    if (row_stride < vocab) return kv_fail(NF_ERR_SHAPE, "the row stride must be at least vocab");
    if (top < 0 || top > kMaxTop || top > vocab)
        return kv_fail(NF_ERR_UNSUPPORTED, "top must be in [0, %d] and at most vocab", kMaxTop);
    if (!target != !logprob) return kv_fail(NF_ERR_INVALID, "targets and log-probabilities go together");
    if (rows == 0) return NF_OK;
    if (!logits || (top > 0 && (!top_idx || !top_lp))) return kv_fail(NF_ERR_INVALID, "null logits or top pointer");
    if (reinterpret_cast<uintptr_t>(logits) % (logits_type == NF_DTYPE_F32 ? 4 : 2) != 0)
        return kv_fail(NF_ERR_LAYOUT, "logits must be aligned to their type");
    const int64_t need = nf_token_logprobs_workspace(rows, vocab, top);
    if (!work || work_bytes < need)
        return kv_fail(NF_ERR_CAPACITY, "the workspace must hold %lld bytes", static_cast<long long>(need));
    if (reinterpret_cast<uintptr_t>(work) % 16 != 0)
        return kv_fail(NF_ERR_LAYOUT, "the workspace must be 16-byte aligned");
    const cudaError_t e = launch_token_logprobs(logits, logits_type, row_stride, rows, vocab, target, top, logprob,
                                                entropy, top_idx, top_lp, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return kv_fail(NF_ERR_CUDA, "log-probability launch: %s", cudaGetErrorString(e));
    return NF_OK;
}

}  // extern "C"
