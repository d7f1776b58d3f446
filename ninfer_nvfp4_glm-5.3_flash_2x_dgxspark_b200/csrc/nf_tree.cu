// nf_tree.cu -- nf_tree_attention (include/nf_moe.h): attention of a
// sequence's new rows, one token, a chain or a tree, over its cached prefix
// and over one another.
#include "nf_kv.h"

#include "nf_common.cuh"
#include "nf_internal.h"

#include <cmath>

namespace nf {

namespace {

constexpr int64_t kWorkBytes = 256;
constexpr int kStatusBad = NF_DEVERR_BAD_TOKEN;

// One warp per (row, q head); lane l holds dims l D / 32 ...
template <int D>
__global__ void __launch_bounds__(128) tree_attention_kernel(const __grid_constant__ nf_kv_cache c,
                                                             const uint16_t* __restrict__ q, int rows, int nq,
                                                             const int32_t* __restrict__ row_start, int batch,
                                                             const int32_t* __restrict__ prefix,
                                                             const int32_t* __restrict__ cache_seq,
                                                             const uint64_t* __restrict__ mask, int words, float scale,
                                                             uint16_t* __restrict__ out, int32_t* __restrict__ status) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31;
    const int64_t gw = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    if (gw >= static_cast<int64_t>(rows) * nq) return;
    const int r = static_cast<int>(gw / nq), h = static_cast<int>(gw % nq), g = h / (nq / c.kv_heads);
    // the last sequence that starts at or before row r
    int i = -1;
    for (int a = 0; a < batch; ++a)
        if (r >= row_start[a] && r < row_start[a + 1]) i = a;
    if (i < 0) return;
    const int r0 = max(0, row_start[i]), n = min(rows, row_start[i + 1]) - r0;
    const int p0 = prefix[i], sq = cache_seq ? cache_seq[i] : i;
    uint16_t* o = out + gw * D + lane * E;
    if (p0 < 0 || sq < 0 || sq >= c.seqs || n > c.max_context - p0) {
        if (lane == 0 && status) atomicCAS(status, 0, kStatusBad);
        for (int e = 0; e < E; ++e) o[e] = 0x7fc0;
        return;
    }
    float qr[E], acc[E], m = -INFINITY, l = 0.f;
    for (int e = 0; e < E; ++e) {
        qr[e] = bf16_bits_to_f32(q[gw * D + lane * E + e]) * scale;
        acc[e] = 0.f;
    }
    const int64_t base = (static_cast<int64_t>(sq) * c.kv_heads + g) * c.max_context;
    for (int j = 0; j < p0 + n; ++j) {
        if (j >= p0) {
            const int node = j - p0;
            if (mask ? node >= 64 * words || !((mask[static_cast<int64_t>(r) * words + (node >> 6)] >> (node & 63)) & 1)
                     : node > r - r0)
                continue;
        }
        const int64_t at = (base + j) * D + lane * E;
        float s = 0.f, kf[E], vf[E], vs = 1.f;
        for (int e = 0; e < E; ++e) {
            kf[e] = c.kind == NF_KV_BF16 ? bf16_bits_to_f32(static_cast<const uint16_t*>(c.k)[at + e])
                                         : e4m3_to_f32(static_cast<const uint8_t*>(c.k)[at + e]);
            vf[e] = c.kind == NF_KV_BF16 ? bf16_bits_to_f32(static_cast<const uint16_t*>(c.v)[at + e])
                                         : e4m3_to_f32(static_cast<const uint8_t*>(c.v)[at + e]);
            s = __fmaf_rn(qr[e], kf[e], s);
        }
        for (int k = 16; k > 0; k >>= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
        if (c.kind == NF_KV_E4M3) {
            s *= c.k_scale[base + j];
            vs = c.v_scale[base + j];
        }
        const float mn = fmaxf(m, s), corr = m == -INFINITY ? 0.f : expf(m - mn), pr = expf(s - mn);
        m = mn;
        l = l * corr + pr;
        for (int e = 0; e < E; ++e) acc[e] = acc[e] * corr + pr * (vf[e] * vs);
    }
    for (int e = 0; e < E; ++e) o[e] = f32_to_bf16_bits(l == 0.f ? 0.f : acc[e] / l);
}

}  // namespace

cudaError_t launch_tree_attention(const nf_kv_cache& c, const uint16_t* q, int rows, int q_heads,
                                  const int32_t* row_start, int batch, const int32_t* prefix, const int32_t* cache_seq,
                                  const uint64_t* mask, int mask_words, float scale, uint16_t* out, void*,
                                  int32_t* status, cudaStream_t st) {
    if (rows <= 0 || batch <= 0) return cudaSuccess;
    const int64_t warps = static_cast<int64_t>(rows) * q_heads;
    auto kernel = c.head_dim == 128 ? tree_attention_kernel<128> : tree_attention_kernel<64>;
    kernel<<<static_cast<unsigned>((warps + 3) / 4), 128, 0, st>>>(c, q, rows, q_heads, row_start, batch, prefix,
                                                                   cache_seq, mask, mask_words, scale, out, status);
    return cudaGetLastError();
}

}  // namespace nf

using namespace nf;

extern "C" {

int64_t nf_tree_attention_workspace(int head_dim) { return head_dim == 64 || head_dim == 128 ? kWorkBytes : 0; }

int nf_tree_attention(const nf_kv_cache* cache, const uint16_t* q, int rows, int q_heads, const int32_t* row_start,
                      int batch, const int32_t* prefix, const int32_t* cache_seq, const uint64_t* mask, int mask_words,
                      float scale, uint16_t* out, void* work, int64_t work_bytes, int32_t* status, void* stream) {
    kv_clear_error();
    const int st = kv_check_cache(cache);
    if (st != NF_OK) return st;
    if (rows < 0 || batch < 0) return kv_fail(NF_ERR_INVALID, "rows and batch must be >= 0");
    if (q_heads < 1 || q_heads % cache->kv_heads != 0 || q_heads / cache->kv_heads > 128)
        return kv_fail(NF_ERR_SHAPE, "q_heads %d must be a multiple of the %d KV heads, at most 128 for each", q_heads,
                       cache->kv_heads);
    if (static_cast<int64_t>(rows) * q_heads > 0x7fffffffll)
        return kv_fail(NF_ERR_CAPACITY, "rows x q_heads must be below 2^31");
    if (mask && (mask_words < 1 || mask_words > 64)) return kv_fail(NF_ERR_SHAPE, "mask_words must be in [1, 64]");
    if (!std::isfinite(scale)) return kv_fail(NF_ERR_INVALID, "the scale must be finite");
    if (rows == 0 || batch == 0) return NF_OK;
    if (!q || !row_start || !prefix || !out) return kv_fail(NF_ERR_INVALID, "null q, row_start, prefix or output pointer");
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) % 16 != 0 ||
        reinterpret_cast<uintptr_t>(mask) % 8 != 0)
        return kv_fail(NF_ERR_LAYOUT, "q and the output must be 16-byte aligned, the mask 8-byte aligned");
    const int64_t need = nf_tree_attention_workspace(cache->head_dim);
    if (!work || work_bytes < need)
        return kv_fail(NF_ERR_CAPACITY, "the workspace must hold %lld bytes", static_cast<long long>(need));
    if (reinterpret_cast<uintptr_t>(work) % 256 != 0)
        return kv_fail(NF_ERR_LAYOUT, "the workspace must be 256-byte aligned");
    const cudaError_t e = launch_tree_attention(*cache, q, rows, q_heads, row_start, batch, prefix, cache_seq, mask,
                                                mask_words, scale, out, work, status, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return kv_fail(NF_ERR_CUDA, "tree attention launch: %s", cudaGetErrorString(e));
    return NF_OK;
}

}  // extern "C"
