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
#include <type_traits>

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
    if (status == NF_ERR_CUDA) cudaGetLastError();  // told here, and no later launch's failure
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
// kv_write: a CTA per token, half a warp per head in turn; lane l of 16 holds
// the head's dims l D / 16 .. (l + 1) D / 16 - 1.  The bytes of q, k and v are
// the floor; what bounds it is the instructions issued, of which half are per
// head and not per dim, so a warp takes two heads at a time.  The next heads'
// rows are on their way meanwhile, and the angles' sines are taken once per
// token, while the first come in.  A rotated pair lies in a lane (interleaved;
// FULL below), or in two lanes whose distance is the pairs' (halves, when that
// is a whole number of lanes), else it goes through shared memory.
// 8,192 tokens, 32 + 2 x 4 heads of 128, BF16 to E4M3: 43 us, 3.7 TB/s of the
// bytes; exchanging the pairs' dims between lanes it was 51.  Two or three
// heads ahead instead of one: 50.
// ---------------------------------------------------------------------------
constexpr int kWriteWarps = 8;  // at most

__device__ __forceinline__ float half_warp_sum(float v) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// E neighbouring dims as loaded: 4-byte words, of one F32 or two BF16 dims.
template <int W>
__device__ __forceinline__ void load_words(const void* p, uint32_t* w) {
    if (W == 1) {
        w[0] = __ldg(static_cast<const uint32_t*>(p));
    } else if (W == 2) {
        const uint2 v = __ldg(static_cast<const uint2*>(p));
        w[0] = v.x;
        w[W - 1] = v.y;
    } else {
#pragma unroll
        for (int k = 0; k < W / 4; ++k) {
            const uint4 v = __ldg(static_cast<const uint4*>(p) + k);
            w[4 * k] = v.x;
            w[4 * k + 1] = v.y;
            w[4 * k + 2] = v.z;
            w[4 * k + 3] = v.w;
        }
    }
}
template <int E>
__device__ __forceinline__ void store_bf16(uint16_t* dst, const float* x) {
    uint32_t w[E / 2];
#pragma unroll
    for (int e = 0; e < E; e += 2) w[e / 2] = bf16x2_hw(x[e], x[e + 1]);
    if (E == 8) *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[E / 2 - 2], w[E / 2 - 1]);
    else if (E == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[E / 2 - 1]);
    else *reinterpret_cast<uint32_t*>(dst) = w[0];
}

// A lane's dims of a row whose greatest magnitude is `peak` as E4M3 codes;
// returns the row's scale.
template <int E>
__device__ __forceinline__ float quantize_row(float (&y)[E], float peak, uint32_t (&code)[E / 4]) {
    const float scale = peak * (1.f / 448.f);
    if (peak >= 1e-30f && peak <= 1e30f) {
        const float inv = __fdividef(448.f, peak);
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] *= inv;
    } else {  // zeros, where the quotient might overflow, and NaN
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = scale > 0.f || isnan(scale) ? __fdiv_rn(y[e], scale) : 0.f;
    }
#pragma unroll
    for (int e = 0; e < E; e += 4) {
        uint16_t lo, hi;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(y[e + 1]), "f"(y[e]));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(y[e + 3]), "f"(y[e + 2]));
        code[e / 4] = lo | static_cast<uint32_t>(hi) << 16;
    }
    return scale;
}
template <int E>
__device__ __forceinline__ float half_warp_peak(const float (&y)[E]) {
    float peak = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) peak = max_nan(peak, fabsf(y[e]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) peak = max_nan(peak, __shfl_xor_sync(0xffffffffu, peak, o));
    return peak;
}

// FULL: the two halves of all dims rotate with one another.  Then a lane holds
// E / 2 dims of either half, so that its pairs need no exchange.
template <int D, bool BF16, bool FULL>
__global__ void __launch_bounds__(32 * kWriteWarps, 4) kv_write_kernel(
    const __grid_constant__ nf_kv_cache c, const __grid_constant__ nf_rope rope, const void* __restrict__ qkv,
    int slices, int64_t slice_stride, int64_t row_stride, int nq, const float* __restrict__ q_norm,
    const float* __restrict__ k_norm, float eps, const int32_t* __restrict__ pos, const int32_t* __restrict__ seq,
    const int32_t* __restrict__ slot, uint16_t* __restrict__ q_out, int32_t* __restrict__ status) {
    constexpr int E = D / 16, W = BF16 ? E / 2 : E, H = FULL ? E / 2 : E, kSize = BF16 ? 2 : 4;
    const int step = blockDim.x >> 4;  // heads at a time
    __shared__ float2 s_turn[D / 2];  // (cos, sin) of every pair's angle, times the magnitude
    __shared__ float s_row[FULL ? 1 : 2 * kWriteWarps][FULL ? 1 : D];
    const int sub = threadIdx.x >> 4, lane = threadIdx.x & 15;  // which half warp, and the lane in it
    const int nkv = c.kv_heads, heads = nq + 2 * nkv, t = blockIdx.x;
    auto dim = [&](int e) { return (e < H ? 0 : D / 2 - H) + lane * H + e; };  // the lane's e-th
    const uint8_t* row = static_cast<const uint8_t*>(qkv) + (static_cast<int64_t>(t) * row_stride + lane * H) * kSize;
    auto fetch = [&](int64_t at, uint32_t* w) {
        if constexpr (FULL) {
            load_words<W / 2>(row + at * kSize, w);
            load_words<W / 2>(row + (at + D / 2) * kSize, w + W / 2);
        } else {
            load_words<W>(row + at * kSize, w);
        }
    };
    uint32_t next[W];
    auto load = [&](int h) {
        if (h < heads) fetch(static_cast<int64_t>(h) * D, next);
    };
    load(sub < nq ? sub : nq + sub);

    const int p = pos[t], sq = seq ? seq[t] : t, sl = slot ? slot[t] : p;
    const bool ok = p >= 0 && (sl == -1 || (sq >= 0 && sq < c.seqs && sl >= 0 && sl < c.max_context));
    if (!ok && threadIdx.x == 0 && status) atomicCAS(status, 0, kStatusBad);
    const int rd = rope.rotary_dim, half = rd >> 1;
    const bool inter = rope.layout == NF_ROPE_INTERLEAVED;
#pragma unroll 1
    for (int i = threadIdx.x; i < half; i += blockDim.x) {
        // the angle's fraction of a turn, in [-1/2, 1/2)
        const int32_t frac = static_cast<int32_t>((static_cast<uint64_t>(p) * rope.turn[i]) >> 32);
        float s, co;
        sincospif(static_cast<float>(frac) * 4.656612873077393e-10f /* 2^-31 */, &s, &co);
        s_turn[i] = make_float2(co * rope.magnitude, s * rope.magnitude);
    }
    float wq[E], wk[E];  // the norms' weights of the lane's dims
#pragma unroll
    for (int e = 0; e < E; ++e) {
        wq[e] = q_norm ? __ldg(q_norm + dim(e)) : 1.f;
        wk[e] = k_norm ? __ldg(k_norm + dim(e)) : 1.f;
    }
    __syncthreads();
    // the lane's dims' angles, the same in every head; dims behind rd do not turn
    float co[E], si[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int i = dim(e);
        const float2 f = i >= rd ? make_float2(1.f, 0.f) : s_turn[inter ? i >> 1 : i < half ? i : i - half];
        co[e] = f.x;
        si[e] = (inter ? (i & 1) == 0 : i < half) ? -f.y : f.y;  // first a cos - b sin, second b cos + a sin
    }
    const bool near = half % E == 0;  // a pair's second dim lies `half / E` lanes on, at the same place
    const int other = (threadIdx.x & 16) + ((lane * E < half ? lane + half / E : lane - half / E) & 15);
    const int64_t base = sl < 0 ? 0 : static_cast<int64_t>(sq) * nkv * c.max_context + sl;

    auto take = [&](int h, bool in, int following, float (&y)[E]) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const uint32_t w = next[BF16 ? e / 2 : e];
            y[e] = !in ? 0.f : __uint_as_float(!BF16 ? w : (e & 1) ? w & 0xffff0000u : w << 16);
        }
        if (!BF16 && in)
#pragma unroll 1
            for (int k = 1; k < slices; ++k) {
                uint32_t w[W];
                fetch(k * slice_stride + static_cast<int64_t>(h) * D, w);
#pragma unroll
                for (int e = 0; e < E; ++e) y[e] = __fadd_rn(y[e], __uint_as_float(w[BF16 ? 0 : e]));
            }
        load(following);
    };
    auto normalise = [&](float (&y)[E], const float (&w)[E], bool on) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) ss = __fmaf_rn(y[e], y[e], ss);
        ss = half_warp_sum(ss);
        const float inv = rsqrtf(__fmaf_rn(ss, 1.f / D, eps));
        if (on)
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] = __fmul_rn(__fmul_rn(y[e], inv), w[e]);
    };
    auto rotate = [&](float (&y)[E], bool on) {
        if (rd == 0) return;
        float z[E];
        if (FULL) {
#pragma unroll
            for (int e = 0; e < E; ++e) z[e] = y[e < H ? e + H : e - H];
        } else if (inter) {
#pragma unroll
            for (int e = 0; e < E; ++e) z[e] = y[e ^ 1];
        } else if (near) {
#pragma unroll
            for (int e = 0; e < E; ++e) z[e] = __shfl_sync(0xffffffffu, y[e], other);
        } else {
            __syncwarp();
#pragma unroll
            for (int e = 0; e < E; ++e) s_row[FULL ? 0 : sub][FULL ? 0 : lane * E + e] = y[e];
            __syncwarp();
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int i = lane * E + e;
                z[e] = i >= rd ? 0.f : s_row[FULL ? 0 : sub][FULL ? 0 : i < half ? i + half : i - half];
            }
        }
        if (on)
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (FULL || lane * E + e < rd) y[e] = fmaf(z[e], si[e], y[e] * co[e]);
    };
    auto store = [&](uint16_t* dst, const float (&y)[E]) {
        if constexpr (FULL) {
            store_bf16<H>(dst + lane * H, y);
            store_bf16<H>(dst + D / 2 + lane * H, y + H);
        } else {
            store_bf16<E>(dst + lane * E, y);
        }
    };

    // q's heads, then K's and V's; both halves of a warp take the same steps
#pragma unroll 1
    for (int h = sub; h - sub < nq; h += step) {
        const bool in = h < nq;
        float y[E];
        take(h, in, h + step < nq ? h + step : nq + sub, y);
        if (q_norm) normalise(y, wq, true);
        rotate(y, true);
        if (!in) continue;
        if (!ok)
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] = NAN;
        store(q_out + (static_cast<int64_t>(t) * nq + h) * D, y);
    }
#pragma unroll 1
    for (int h = nq + sub; h - sub < heads; h += step) {
        const bool in = h < heads, is_k = h < nq + nkv;
        float y[E];
        take(h, in, h + step, y);
        if (__any_sync(0xffffffffu, is_k)) {
            if (k_norm) normalise(y, wk, is_k);
            rotate(y, is_k);
        }
        float peak = 0.f;
        if (c.kind == NF_KV_E4M3) peak = half_warp_peak<E>(y);
        if (!in || !ok || sl < 0) continue;
        const int64_t r = base + static_cast<int64_t>(is_k ? h - nq : h - nq - nkv) * c.max_context;
        if (c.kind == NF_KV_BF16) {
            store(static_cast<uint16_t*>(is_k ? c.k : c.v) + r * D, y);
            continue;
        }
        uint32_t code[E / 4];
        const float scale = quantize_row<E>(y, peak, code);
        uint8_t* dst = static_cast<uint8_t*>(is_k ? c.k : c.v) + r * D + lane * H;
        if constexpr (FULL && E == 8) {
            *reinterpret_cast<uint32_t*>(dst) = code[0];
            *reinterpret_cast<uint32_t*>(dst + D / 2) = code[E / 4 - 1];
        } else if constexpr (FULL) {
            *reinterpret_cast<uint16_t*>(dst) = static_cast<uint16_t>(code[0]);
            *reinterpret_cast<uint16_t*>(dst + D / 2) = static_cast<uint16_t>(code[0] >> 16);
        } else if constexpr (E == 8) {
            *reinterpret_cast<uint2*>(dst) = make_uint2(code[0], code[E / 4 - 1]);
        } else {
            *reinterpret_cast<uint32_t*>(dst) = code[0];
        }
        if (lane == 0) (is_k ? c.k_scale : c.v_scale)[r] = scale;
    }
}

// A loaded history's rows, half a warp each.
template <int D>
__global__ void __launch_bounds__(256) kv_quantize_kernel(const uint16_t* __restrict__ x, int64_t n,
                                                          uint8_t* __restrict__ codes, float* __restrict__ scale) {
    constexpr int E = D / 16;
    const int lane = threadIdx.x & 15;
    const int64_t r = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 4;
    float y[E];
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = r < n ? bf16_bits_to_f32(x[r * D + lane * E + e]) : 0.f;
    uint32_t code[E / 4];
    const float s = quantize_row<E>(y, half_warp_peak<E>(y), code);
    if (r >= n) return;
#pragma unroll
    for (int e = 0; e < E / 4; ++e) *reinterpret_cast<uint32_t*>(codes + r * D + lane * E + 4 * e) = code[e];
    if (lane == 0) scale[r] = s;
}

// The same view of a batch as the attention's: row_start is clamped to
// [0, rows], and a sequence is refused as a whole, so that none of its rows is
// written when one of them, or its position, lies outside.
__global__ void __launch_bounds__(128) kv_places_kernel(int rows, int L, const int32_t* __restrict__ row_start, int batch,
                                                        const int32_t* __restrict__ prefix,
                                                        const int32_t* __restrict__ depth, int32_t* __restrict__ seq,
                                                        int32_t* __restrict__ slot, int32_t* __restrict__ pos) {
    const int r = blockIdx.x * blockDim.x + threadIdx.x;
    if (r >= rows) return;
    auto start = [&](int i) { return min(max(row_start[i], 0), rows); };
    int lo = 0, hi = batch;  // the last sequence that starts at or before r
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (start(mid) <= r) lo = mid;
        else hi = mid;
    }
    const int first = start(lo), n = start(lo + 1) - first, j = r - first, p0 = prefix[lo];
    const bool in = j >= 0 && j < n;
    bool bad = p0 < 0 || p0 > L - n;
    if (in && depth)
#pragma unroll 4
        for (int k = 0; k < n; ++k) {
            const int64_t p = static_cast<int64_t>(p0) + depth[first + k];
            bad |= p < 0 || p > 0x7fffffff;
        }
    // the write refuses these places
    seq[r] = lo;
    slot[r] = !in ? -1 : bad ? 0x7fffffff : p0 + j;
    pos[r] = !in ? 0 : bad ? -1 : p0 + (depth ? depth[r] : j);
}

// ---------------------------------------------------------------------------
// kv_accept: the path rises, so row j moves down to a slot that no later move
// reads (path[j'] >= j' > j), and every 16-byte column of a row can be moved
// by one thread in path order.  Bound by the latency of loads and stores at
// scattered rows: every (layer, sequence) has its own CTA.  200 sequences in
// 46 layers, E4M3 rows of 128 bytes: 24.6 us, 2.9 TB/s of the moved bytes.
// ---------------------------------------------------------------------------
constexpr int kAcceptLayers = 64;  // caches per launch
struct AcceptCaches {
    uint8_t* k[kAcceptLayers];
    uint8_t* v[kAcceptLayers];
    float* ks[kAcceptLayers];
    float* vs[kAcceptLayers];
};

// One thread's column of n rows to their places, four loads ahead of the stores (200 sequences x 46 layers: 24.6 us, with
// eight 28.7, whose registers leave an SM fewer CTAs).
template <typename T>
__device__ __forceinline__ void move_rows(uint8_t* base, int64_t pitch, const int32_t* __restrict__ path, int n) {
#pragma unroll 1
    for (int j0 = 0; j0 < n; j0 += 4) {
        T v[4];
        bool go[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int from = j0 + k < n ? path[j0 + k] : j0 + k;
            go[k] = from != j0 + k;
            if (go[k]) v[k] = *reinterpret_cast<const T*>(base + from * pitch);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (go[k]) *reinterpret_cast<T*>(base + (j0 + k) * pitch) = v[k];
    }
}

__global__ void __launch_bounds__(128) kv_accept_kernel(const __grid_constant__ AcceptCaches a, int e4m3, int seqs,
                                                        int nkv, int L, int row_bytes, int first,
                                                        const int32_t* __restrict__ prefix,
                                                        const int32_t* __restrict__ path, int max_path,
                                                        const int32_t* __restrict__ path_len,
                                                        const int32_t* __restrict__ cache_seq,
                                                        int32_t* __restrict__ status) {
    const int i = blockIdx.y, layer = blockIdx.z;
    const int n = path_len[i], p0 = prefix[i], sq = cache_seq ? cache_seq[i] : first + i;
    const int32_t* pa = path + static_cast<int64_t>(i) * max_path;
    bool ok = n >= 0 && n <= max_path && p0 >= 0 && p0 <= L && sq >= 0 && sq < seqs;
    if (ok) {
        int last = -1;
#pragma unroll 8
        for (int j = 0; j < n; ++j) {
            const int at = pa[j];
            ok &= at > last && at < L - p0;
            last = at;
        }
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
            move_rows<uint4>(base, row_bytes, pa, n);
        } else {
            move_rows<float>(reinterpret_cast<uint8_t*>(((u & 1) ? a.vs : a.ks)[layer] + row), 4, pa, n);
        }
    }
}

}  // namespace

cudaError_t launch_kv_write(const nf_kv_cache& c, const nf_rope& rope, const void* qkv, int qkv_type,
                            int64_t row_stride, int tokens, int q_heads, const float* q_norm, const float* k_norm,
                            float eps, const int32_t* pos, const int32_t* seq, const int32_t* slot, uint16_t* q,
                            int32_t* status, cudaStream_t st, int slices, int64_t slice_stride) {
    if (tokens <= 0) return cudaSuccess;
    const bool bf16 = qkv_type == NF_DTYPE_BF16;
    const bool full = rope.rotary_dim == c.head_dim && rope.layout == NF_ROPE_HALF;
    auto pick = [&](auto d, auto f) {
        return bf16 ? kv_write_kernel<decltype(d)::value, true, decltype(f)::value>
                    : kv_write_kernel<decltype(d)::value, false, decltype(f)::value>;
    };
    using Wide = std::integral_constant<int, 128>;
    using Narrow = std::integral_constant<int, 64>;
    auto kernel = c.head_dim == 128 ? (full ? pick(Wide(), std::true_type()) : pick(Wide(), std::false_type()))
                                    : (full ? pick(Narrow(), std::true_type()) : pick(Narrow(), std::false_type()));
    // Few tokens: more warps share a token's heads; many: fewer, so that less of the time goes to what is done once per
    // token.  Measured with 8, 4, 2 warps (us between events, 40 heads of 128, BF16 rows): 64 tokens 9.2 10.2 13.2;
    // 600: 13.3 12.3 14.4; 1,000: 15.3 13.3 15.4; 2,000: 22.5 19.4 17.5; 8,192: 64.5 50.2 48.0 (one warp: 48.2).
    const int warps = tokens <= 2 * 148 ? kWriteWarps : tokens <= 1000 ? 4 : 2;
    kernel<<<static_cast<unsigned>(tokens), 32 * warps, 0, st>>>(c, rope, qkv, slices, slice_stride, row_stride, q_heads,
                                                                 q_norm, k_norm, eps, pos, seq, slot, q, status);
    return cudaGetLastError();
}

cudaError_t launch_kv_quantize(const uint16_t* x, int64_t n, int head_dim, uint8_t* codes, float* scale, cudaStream_t st) {
    if (n <= 0) return cudaSuccess;
    const unsigned grid = static_cast<unsigned>((n + 15) / 16);
    if (head_dim == 128) kv_quantize_kernel<128><<<grid, 256, 0, st>>>(x, n, codes, scale);
    else kv_quantize_kernel<64><<<grid, 256, 0, st>>>(x, n, codes, scale);
    return cudaGetLastError();
}

cudaError_t launch_kv_places(int rows, int max_context, const int32_t* row_start, int batch, const int32_t* prefix, const int32_t* depth,
                             int32_t* seq, int32_t* slot, int32_t* pos, cudaStream_t st) {
    if (rows <= 0) return cudaSuccess;
    kv_places_kernel<<<(rows + 127) / 128, 128, 0, st>>>(rows, max_context, row_start, batch, prefix, depth, seq, slot, pos);
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
                                                              c.max_context, row_bytes, i0, prefix + i0,
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
    if (layers > 0 && static_cast<int64_t>(caches[0].kv_heads) * 2 * (caches[0].head_dim / 8 + 1) > 0x7fffffffll)
        return kv_fail(NF_ERR_CAPACITY, "a position's rows of %d KV heads: 16-byte pieces must be below 2^31", caches[0].kv_heads);
    if (layers == 0 || batch == 0 || max_path == 0) return NF_OK;
    if (!prefix || !path || !path_len) return kv_fail(NF_ERR_INVALID, "null prefix, path or length pointer");
    const cudaError_t e = launch_kv_accept(caches, layers, prefix, path, max_path, path_len, cache_seq, batch, status,
                                           static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return kv_fail(NF_ERR_CUDA, "cache move launch: %s", cudaGetErrorString(e));
    return NF_OK;
}

}  // extern "C"
