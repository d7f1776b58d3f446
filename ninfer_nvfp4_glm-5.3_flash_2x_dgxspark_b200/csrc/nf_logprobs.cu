// nf_logprobs.cu -- nf_token_logprobs (include/nf_moe.h): log-probability of
// a given token, entropy and the greatest logits of every row.
#include "nf_kv.h"

#include "nf_common.cuh"
#include "nf_internal.h"

#include <cmath>

namespace nf {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTop = 32;

// A logit's place in the order of the top tokens: greater logits first, -0
// and +0 equal, a NaN behind everything; the lower index first among equals.
__device__ __forceinline__ uint64_t order_key(float x, int64_t index) {
    uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);
    b = isnan(x) ? 0u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return (static_cast<uint64_t>(b) << 32) | (0xffffffffu - static_cast<uint32_t>(index));
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

// One CTA per row; the maximum, the sums, then one pass per top token.
template <bool BF16>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(const void* __restrict__ logits, int64_t stride,
                                                                  int64_t vocab, const int32_t* __restrict__ target,
                                                                  int top, float* __restrict__ logprob,
                                                                  float* __restrict__ entropy,
                                                                  int32_t* __restrict__ top_idx,
                                                                  float* __restrict__ top_lp) {
    __shared__ uint64_t s_u[kThreads / 32];
    __shared__ float s_f[kThreads / 32];
    const int64_t row = blockIdx.x;
    const void* x = static_cast<const uint8_t*>(logits) + row * stride * (BF16 ? 2 : 4);
    auto fmaxnan = [](float a, float b) { return isnan(a) || isnan(b) ? NAN : fmaxf(a, b); };
    auto add = [](float a, float b) { return a + b; };
    float m = -INFINITY;
    for (int64_t i = threadIdx.x; i < vocab; i += kThreads) m = fmaxnan(m, load_logit<BF16>(x, i));
    m = block_reduce(m, s_f, fmaxnan);
    float s = 0.f, t = 0.f;
    for (int64_t i = threadIdx.x; i < vocab; i += kThreads) {
        const float d = load_logit<BF16>(x, i) - m, e = expf(d);
        s += e;
        t += e > 0.f ? e * d : e * 0.f;
    }
    s = block_reduce(s, s_f, add);
    t = block_reduce(t, s_f, add);
    const float ls = isinf(m) ? NAN : logf(s);
    if (threadIdx.x == 0) {
        if (logprob) {
            const int32_t id = target[row];
            logprob[row] = id >= 0 && id < vocab ? load_logit<BF16>(x, id) - m - ls : NAN;
        }
        if (entropy) entropy[row] = ls - t / s;
    }
    uint64_t last = ~0ull;
    for (int k = 0; k < top; ++k) {
        uint64_t best = 0;
        for (int64_t i = threadIdx.x; i < vocab; i += kThreads) {
            const uint64_t u = order_key(load_logit<BF16>(x, i), i);
            if (u < last && u > best) best = u;
        }
        best = block_reduce(best, s_u, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
        if (threadIdx.x == 0) {
            const int32_t id = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(best));
            top_idx[row * top + k] = id;
            top_lp[row * top + k] = load_logit<BF16>(x, id) - m - ls;
        }
        last = best;
    }
}

}  // namespace

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
    auto kernel = logits_type == NF_DTYPE_BF16 ? token_logprobs_kernel<true> : token_logprobs_kernel<false>;
    kernel<<<rows, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(logits, row_stride, vocab, target, top, logprob,
                                                                    entropy, top_idx, top_lp);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return kv_fail(NF_ERR_CUDA, "log-probability launch: %s", cudaGetErrorString(e));
    return NF_OK;
}

}  // extern "C"
