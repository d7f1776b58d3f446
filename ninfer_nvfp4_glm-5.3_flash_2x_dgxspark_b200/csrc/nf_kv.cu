// nf_kv.cu -- the KV cache's side of a drafted-token step (include/nf_moe.h):
// nf_rope_init, nf_kv_write and nf_kv_accept, and the checks the section's
// entry points share.
#include "nf_kv.h"

#include "nf_common.cuh"
#include "nf_internal.h"

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>

namespace nf {

namespace {

thread_local char g_kv_error[512] = "";

constexpr int kStatusBad = NF_DEVERR_BAD_TOKEN;  // what *status_dev becomes

}  // namespace

int kv_fail(int status, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_kv_error, sizeof(g_kv_error), fmt, ap);
    va_end(ap);
    return status;
}

void kv_clear_error() { g_kv_error[0] = '\0'; }

int kv_check_cache(const nf_kv_cache* c) {
    if (!c) return kv_fail(NF_ERR_INVALID, "null cache");
    if (c->kind != NF_KV_BF16 && c->kind != NF_KV_E4M3) return kv_fail(NF_ERR_INVALID, "unknown cache kind %d", c->kind);
    if (c->head_dim != 64 && c->head_dim != 128)
        return kv_fail(NF_ERR_UNSUPPORTED, "cache head_dim must be 64 or 128, not %d", c->head_dim);
    if (c->seqs < 1 || c->kv_heads < 1 || c->max_context < 1 || c->max_context > 1 << 30 ||
        static_cast<int64_t>(c->seqs) * c->kv_heads > 0x7fffffffll)
        return kv_fail(NF_ERR_SHAPE, "cache shape [%d][%d][%d]", c->seqs, c->kv_heads, c->max_context);
    if (!c->k || !c->v) return kv_fail(NF_ERR_INVALID, "null cache pointer");
    if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) % 16 != 0)
        return kv_fail(NF_ERR_LAYOUT, "cache keys and values must be 16-byte aligned");
    if (c->kind == NF_KV_E4M3) {
        if (!c->k_scale || !c->v_scale) return kv_fail(NF_ERR_INVALID, "an E4M3 cache needs its scales");
        if ((reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale)) % 4 != 0)
            return kv_fail(NF_ERR_LAYOUT, "cache scales must be 4-byte aligned");
    } else if (c->k_scale || c->v_scale) {
        return kv_fail(NF_ERR_INVALID, "a BF16 cache has no scales");
    }
    return NF_OK;
}

namespace {

// ---------------------------------------------------------------------------
// kv_write: one warp per (token, head); lane l holds the head's dims
// l D / 32 .. (l + 1) D / 32 - 1, and a rotated pair's partner comes through
// the warp's shared row.
// ---------------------------------------------------------------------------
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// max over the warp that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

template <int D>
__global__ void __launch_bounds__(128) kv_write_kernel(const __grid_constant__ nf_kv_cache c,
                                                       const __grid_constant__ nf_rope rope,
                                                       const void* __restrict__ qkv, int bf16_in, int64_t row_stride,
                                                       int tokens, int nq, const float* __restrict__ q_norm,
                                                       const float* __restrict__ k_norm, float eps,
                                                       const int32_t* __restrict__ pos, const int32_t* __restrict__ seq,
                                                       const int32_t* __restrict__ slot, uint16_t* __restrict__ q_out,
                                                       int32_t* __restrict__ status) {
    constexpr int E = D / 32;
    __shared__ float s_row[4][D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int nkv = c.kv_heads, heads = nq + 2 * nkv;
    const int64_t gw = static_cast<int64_t>(blockIdx.x) * 4 + warp;
    if (gw >= static_cast<int64_t>(tokens) * heads) return;
    const int t = static_cast<int>(gw / heads), h = static_cast<int>(gw % heads);
    const int p = pos[t], sq = seq ? seq[t] : t, sl = slot ? slot[t] : p;
    const bool ok = p >= 0 && (sl == -1 || (sq >= 0 && sq < c.seqs && sl >= 0 && sl < c.max_context));
    if (!ok && lane == 0 && status) atomicCAS(status, 0, kStatusBad);
    const bool is_q = h < nq, is_k = !is_q && h < nq + nkv;
    if (!is_q && (!ok || sl < 0)) return;

    float x[E];
    const int64_t at = static_cast<int64_t>(t) * row_stride + static_cast<int64_t>(h) * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e)
        x[e] = bf16_in ? bf16_bits_to_f32(static_cast<const uint16_t*>(qkv)[at + e]) : static_cast<const float*>(qkv)[at + e];
    if (is_q || is_k) {
        const float* nw = is_q ? q_norm : k_norm;
        if (nw) {
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) ss = __fmaf_rn(x[e], x[e], ss);
            ss = warp_sum(ss);
            const float inv = __fdiv_rn(1.f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, static_cast<float>(D)), eps)));
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = __fmul_rn(__fmul_rn(x[e], inv), nw[lane * E + e]);
        }
        const int rd = rope.rotary_dim, half = rd >> 1;
        if (rd > 0) {
#pragma unroll
            for (int e = 0; e < E; ++e) s_row[warp][lane * E + e] = x[e];
            __syncwarp();
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int i = lane * E + e;
                if (i >= rd) continue;
                const bool inter = rope.layout == NF_ROPE_INTERLEAVED;
                const int pair = inter ? i >> 1 : (i < half ? i : i - half);
                const bool first = inter ? (i & 1) == 0 : i < half;
                const float other = s_row[warp][inter ? i ^ 1 : (first ? i + half : i - half)];
                // the angle's fraction of a turn, in [-1/2, 1/2)
                const int32_t frac = static_cast<int32_t>((static_cast<uint64_t>(p) * rope.turn[pair]) >> 32);
                float s, co;
                sincospif(static_cast<float>(frac) * 4.656612873077393e-10f /* 2^-31 */, &s, &co);
                s *= rope.magnitude;
                co *= rope.magnitude;
                x[e] = first ? x[e] * co - other * s : other * s + x[e] * co;
            }
        }
    }
    if (is_q) {
        uint16_t* dst = q_out + (static_cast<int64_t>(t) * nq + h) * D + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) dst[e] = ok ? f32_to_bf16_bits(x[e]) : 0x7fc0;
        return;
    }
    const int g = is_k ? h - nq : h - nq - nkv;
    const int64_t row = (static_cast<int64_t>(sq) * nkv + g) * c.max_context + sl;
    if (c.kind == NF_KV_BF16) {
        uint16_t* dst = static_cast<uint16_t*>(is_k ? c.k : c.v) + row * D + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) dst[e] = f32_to_bf16_bits(x[e]);
        return;
    }
    float peak = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) peak = max_nan(peak, fabsf(x[e]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) peak = max_nan(peak, __shfl_xor_sync(0xffffffffu, peak, o));
    const float scale = __fdiv_rn(peak, 448.f);
    uint8_t* dst = static_cast<uint8_t*>(is_k ? c.k : c.v) + row * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) dst[e] = static_cast<uint8_t>(e4m3_hw(scale > 0.f ? __fdiv_rn(x[e], scale) : 0.f));
    if (lane == 0) (is_k ? c.k_scale : c.v_scale)[row] = scale;
}

// ---------------------------------------------------------------------------
// kv_accept: the path rises, so row j moves down to a slot that no later move
// reads (path[j'] >= j' > j), and every 16-byte column of a row can be moved
// by one thread in path order.
// ---------------------------------------------------------------------------
constexpr int kAcceptLayers = 64;  // caches per launch
struct AcceptCaches {
    uint8_t* k[kAcceptLayers];
    uint8_t* v[kAcceptLayers];
    float* ks[kAcceptLayers];
    float* vs[kAcceptLayers];
};

__global__ void __launch_bounds__(128) kv_accept_kernel(const __grid_constant__ AcceptCaches a, int e4m3, int seqs,
                                                        int nkv, int L, int row_bytes,
                                                        const int32_t* __restrict__ prefix,
                                                        const int32_t* __restrict__ path, int max_path,
                                                        const int32_t* __restrict__ path_len,
                                                        const int32_t* __restrict__ cache_seq,
                                                        int32_t* __restrict__ status) {
    const int i = blockIdx.y, layer = blockIdx.z;
    const int n = path_len[i], p0 = prefix[i], sq = cache_seq ? cache_seq[i] : i;
    const int32_t* pa = path + static_cast<int64_t>(i) * max_path;
    bool ok = n >= 0 && n <= max_path && p0 >= 0 && p0 <= L && sq >= 0 && sq < seqs;
    for (int j = 0, last = -1; ok && j < n; ++j) {
        ok = pa[j] > last && pa[j] < L - p0;
        last = pa[j];
    }
    if (!ok) {
        if (status && threadIdx.x == 0) atomicCAS(status, 0, kStatusBad);
        return;
    }
    // a thread per (head, k or v, 16-byte column), then per (head, k or v) scale
    const int cols = row_bytes / 16, pieces = nkv * 2 * cols, scales = e4m3 ? nkv * 2 : 0;
    for (int w = blockIdx.x * blockDim.x + threadIdx.x; w < pieces + scales; w += gridDim.x * blockDim.x) {
        const int u = w < pieces ? w / cols : w - pieces;
        const int g = u >> 1;
        const int64_t row = (static_cast<int64_t>(sq) * nkv + g) * L + p0;
        if (w < pieces) {
            uint8_t* base = ((u & 1) ? a.v : a.k)[layer] + row * row_bytes + (w % cols) * 16;
            for (int j = 0; j < n; ++j)
                *reinterpret_cast<uint4*>(base + static_cast<int64_t>(j) * row_bytes) =
                    *reinterpret_cast<const uint4*>(base + static_cast<int64_t>(pa[j]) * row_bytes);
        } else {
            float* base = ((u & 1) ? a.vs : a.ks)[layer] + row;
            for (int j = 0; j < n; ++j) base[j] = base[pa[j]];
        }
    }
}

}  // namespace

cudaError_t launch_kv_write(const nf_kv_cache& c, const nf_rope& rope, const void* qkv, int qkv_type,
                            int64_t row_stride, int tokens, int q_heads, const float* q_norm, const float* k_norm,
                            float eps, const int32_t* pos, const int32_t* seq, const int32_t* slot, uint16_t* q,
                            int32_t* status, cudaStream_t st) {
    if (tokens <= 0) return cudaSuccess;
    const int64_t warps = static_cast<int64_t>(tokens) * (q_heads + 2 * c.kv_heads);
    const int bf16 = qkv_type == NF_DTYPE_BF16;
    auto kernel = c.head_dim == 128 ? kv_write_kernel<128> : kv_write_kernel<64>;
    kernel<<<static_cast<unsigned>((warps + 3) / 4), 128, 0, st>>>(c, rope, qkv, bf16, row_stride, tokens, q_heads,
                                                                   q_norm, k_norm, eps, pos, seq, slot, q, status);
    return cudaGetLastError();
}

cudaError_t launch_kv_accept(const nf_kv_cache* caches, int layers, const int32_t* prefix, const int32_t* path,
                             int max_path, const int32_t* path_len, const int32_t* cache_seq, int batch,
                             int32_t* status, cudaStream_t st) {
    if (layers <= 0 || batch <= 0 || max_path <= 0) return cudaSuccess;
    const nf_kv_cache& c = caches[0];
    const int row_bytes = c.head_dim * (c.kind == NF_KV_E4M3 ? 1 : 2);
    const int64_t work = static_cast<int64_t>(c.kv_heads) * 2 * (row_bytes / 16 + (c.kind == NF_KV_E4M3));
    const unsigned gx = static_cast<unsigned>(std::min<int64_t>((work + 127) / 128, 1 << 16));
    for (int l0 = 0; l0 < layers; l0 += kAcceptLayers) {
        const int n = std::min(kAcceptLayers, layers - l0);
        AcceptCaches a{};
        for (int l = 0; l < n; ++l) {
            a.k[l] = static_cast<uint8_t*>(caches[l0 + l].k);
            a.v[l] = static_cast<uint8_t*>(caches[l0 + l].v);
            a.ks[l] = caches[l0 + l].k_scale;
            a.vs[l] = caches[l0 + l].v_scale;
        }
        for (int i0 = 0; i0 < batch; i0 += 65535) {
            const int nb = std::min(65535, batch - i0);
            kv_accept_kernel<<<dim3(gx, nb, n), 128, 0, st>>>(a, c.kind == NF_KV_E4M3, c.seqs, c.kv_heads,
                                                              c.max_context, row_bytes, prefix + i0,
                                                              path + static_cast<int64_t>(i0) * max_path, max_path,
                                                              path_len + i0, cache_seq ? cache_seq + i0 : nullptr, status);
            const cudaError_t e = cudaGetLastError();
            if (e != cudaSuccess) return e;
        }
    }
    return cudaSuccess;
}

}  // namespace nf

using namespace nf;

extern "C" {

const char* nf_kv_last_error(void) { return g_kv_error; }

int nf_rope_init(nf_rope* out, int head_dim, int rotary_dim, int layout, double theta, int scaling, double factor,
                 double original_context, double fast, double slow) {
    kv_clear_error();
    if (!out) return kv_fail(NF_ERR_INVALID, "null rotary table");
    if (head_dim != 64 && head_dim != 128)
        return kv_fail(NF_ERR_UNSUPPORTED, "rotary head_dim must be 64 or 128, not %d", head_dim);
    if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 2 != 0)
        return kv_fail(NF_ERR_SHAPE, "rotary_dim must be even and in [0, head_dim]");
    if (layout != NF_ROPE_HALF && layout != NF_ROPE_INTERLEAVED)
        return kv_fail(NF_ERR_INVALID, "unknown rotary layout %d", layout);
    if (scaling != NF_ROPE_PLAIN && scaling != NF_ROPE_LINEAR && scaling != NF_ROPE_YARN)
        return kv_fail(NF_ERR_INVALID, "unknown rotary scaling %d", scaling);
    if (!(theta > 0.0) || !std::isfinite(theta)) return kv_fail(NF_ERR_INVALID, "rotary theta must be finite and > 0");
    if (scaling != NF_ROPE_PLAIN && (!(factor >= 1.0) || !std::isfinite(factor)))
        return kv_fail(NF_ERR_INVALID, "rotary factor must be finite and >= 1");
    if (scaling == NF_ROPE_YARN && (!(original_context > 0.0) || !std::isfinite(original_context) || !(fast > slow) ||
                                    !std::isfinite(fast) || !std::isfinite(slow)))
        return kv_fail(NF_ERR_INVALID, "YaRN needs original_context > 0 and fast > slow");
    *out = nf_rope{};
    out->head_dim = head_dim;
    out->rotary_dim = rotary_dim;
    out->layout = layout;
    out->magnitude = scaling == NF_ROPE_YARN ? static_cast<float>(0.1 * std::log(factor) + 1.0) : 1.f;
    const long double two_pi = 6.283185307179586476925286766559L;
    for (int i = 0; i < rotary_dim / 2; ++i) {
        long double f = powl(static_cast<long double>(theta), -2.0L * i / rotary_dim);
        if (scaling == NF_ROPE_LINEAR) f /= factor;
        if (scaling == NF_ROPE_YARN) {
            const long double r = original_context * f / two_pi;
            const long double g = std::min(1.0L, std::max(0.0L, (r - slow) / (static_cast<long double>(fast) - slow)));
            f = g * f + (1.0L - g) * f / factor;
        }
        const long double turn = f / two_pi;                      // a whole turn more changes nothing
        const long double frac = ldexpl(turn - floorl(turn), 64);  // [0, 2^64]
        out->turn[i] = frac >= 18446744073709551615.0L ? 0 : static_cast<uint64_t>(frac + 0.5L);
    }
    return NF_OK;
}

int nf_kv_write(const nf_kv_cache* cache, const nf_rope* rope, const void* qkv, int qkv_type, int64_t row_stride,
                int tokens, int q_heads, const float* q_norm, const float* k_norm, float norm_eps, const int32_t* pos,
                const int32_t* seq, const int32_t* slot, uint16_t* q, int32_t* status, void* stream) {
    kv_clear_error();
    const int st = kv_check_cache(cache);
    if (st != NF_OK) return st;
    if (!rope) return kv_fail(NF_ERR_INVALID, "null rotary table");
    if (rope->head_dim != cache->head_dim || rope->rotary_dim < 0 || rope->rotary_dim > rope->head_dim ||
        rope->rotary_dim % 2 != 0)
        return kv_fail(NF_ERR_SHAPE, "rotary table of head_dim %d for a cache of head_dim %d", rope->head_dim,
                       cache->head_dim);
    if (rope->layout != NF_ROPE_HALF && rope->layout != NF_ROPE_INTERLEAVED)
        return kv_fail(NF_ERR_INVALID, "unknown rotary layout %d", rope->layout);
    if (qkv_type != NF_DTYPE_F32 && qkv_type != NF_DTYPE_BF16)
        return kv_fail(NF_ERR_INVALID, "unknown qkv type %d", qkv_type);
    if (tokens < 0) return kv_fail(NF_ERR_INVALID, "tokens must be >= 0");
    if (q_heads < 1 || q_heads > 1 << 16) return kv_fail(NF_ERR_SHAPE, "q_heads must be in [1, 65536]");
    const int64_t heads = q_heads + 2ll * cache->kv_heads;
    if (static_cast<int64_t>(tokens) * heads > 0x7fffffffll)
        return kv_fail(NF_ERR_CAPACITY, "tokens x heads must be below 2^31");
    if (row_stride < heads * cache->head_dim)
        return kv_fail(NF_ERR_SHAPE, "qkv row stride %lld is below the row's %lld elements",
                       static_cast<long long>(row_stride), static_cast<long long>(heads * cache->head_dim));
    const int size = qkv_type == NF_DTYPE_F32 ? 4 : 2;
    if (row_stride * size % 16 != 0 || reinterpret_cast<uintptr_t>(qkv) % 16 != 0 || reinterpret_cast<uintptr_t>(q) % 16 != 0)
        return kv_fail(NF_ERR_LAYOUT, "qkv rows and q must be 16-byte aligned");
    if (!(norm_eps >= 0.f)) return kv_fail(NF_ERR_INVALID, "norm_eps must be >= 0");
    if (tokens == 0) return NF_OK;
    if (!qkv || !pos || !q) return kv_fail(NF_ERR_INVALID, "null qkv, position or q pointer");
    const cudaError_t e = launch_kv_write(*cache, *rope, qkv, qkv_type, row_stride, tokens, q_heads, q_norm, k_norm,
                                          norm_eps, pos, seq, slot, q, status, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return kv_fail(NF_ERR_CUDA, "cache write launch: %s", cudaGetErrorString(e));
    return NF_OK;
}

int nf_kv_accept(const nf_kv_cache* caches, int layers, const int32_t* prefix, const int32_t* path, int max_path,
                 const int32_t* path_len, const int32_t* cache_seq, int batch, int32_t* status, void* stream) {
    kv_clear_error();
    if (layers < 0 || batch < 0 || max_path < 0)
        return kv_fail(NF_ERR_INVALID, "layers, batch and max_path must be >= 0");
    if (layers > 0 && !caches) return kv_fail(NF_ERR_INVALID, "null cache");
    for (int l = 0; l < layers; ++l) {
        const int st = kv_check_cache(caches + l);
        if (st != NF_OK) return st;
        if (caches[l].kind != caches[0].kind || caches[l].seqs != caches[0].seqs ||
            caches[l].kv_heads != caches[0].kv_heads || caches[l].max_context != caches[0].max_context ||
            caches[l].head_dim != caches[0].head_dim)
            return kv_fail(NF_ERR_SHAPE, "the cache of layer %d has another kind or shape than layer 0's", l);
    }
    if (layers == 0 || batch == 0 || max_path == 0) return NF_OK;
    if (!prefix || !path || !path_len) return kv_fail(NF_ERR_INVALID, "null prefix, path or length pointer");
    const cudaError_t e = launch_kv_accept(caches, layers, prefix, path, max_path, path_len, cache_seq, batch, status,
                                           static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return kv_fail(NF_ERR_CUDA, "cache move launch: %s", cudaGetErrorString(e));
    return NF_OK;
}

}  // extern "C"
