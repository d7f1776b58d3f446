// nf_tree_few.cu -- nf_tree_attention's kernel for few rows of a sequence and
// KV head (decode, and trees of a node or two): warp-level tensor-core tiles
// of 16 rows.
//
// The work is the cache's bytes: 16 rows do 32 (BF16) or 64 (E4M3) flops a
// byte, an eighth of what the tensor cores could.  So the keys only have to
// stream: one warp issues TMA tiles of 64 keys into a ring, eight warps take
// 16 keys of a tile each (four warps every other tile), with their own running
// maximum, sum and output in registers, and join at the part's end.  E4M3
// codes become F16 in registers, one conversion for two codes and nothing
// written back to shared memory; q's rows are brought into F16's range by a
// power of two, and so are the probabilities times the values' scales (see
// `ref` below).
#include "nf_tree.cuh"

#include <cmath>

namespace nf {

namespace {

constexpr int kKeys = 64;     // keys per tile
constexpr int kWarps = 8;     // consuming warps
constexpr int kThreads = 32 * (kWarps + 1);

template <int D, bool FP8>
struct Geo {
    static constexpr int kTileBytes = kKeys * D * (FP8 ? 1 : 2);  // K or V
    static constexpr int kStages = FP8 ? 8 : 4;
    static constexpr int kOutAt = kStages * 2 * kTileBytes;             // [warp][16][D] floats
    static constexpr int kMlAt = kOutAt + kWarps * kFewRows * D * 4;    // [warp][16] (m, l)
    static constexpr int kPartAt = kMlAt + kWarps * kFewRows * 8;
    static constexpr int kBarAt = kPartAt + kParts * static_cast<int>(sizeof(Part));
    static constexpr int kSmem = 1024 + kBarAt + (2 * kStages + 2 * kParts + 2) * 8 + 16;
};

// d = a (16 x 16, row) * b (16 x 8, col) + d, F16 in, F32 accumulate
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// Clears the 16-bit halves of a pair of keys (k, k + 1) that lie behind the
// sequence, or that are not finite in a drafted row (which is noted).
template <bool FP8>
__device__ __forceinline__ uint32_t clean(uint32_t v, int k, int node, int end, bool& bad) {
    constexpr uint32_t kExp = FP8 ? 0x7c00u : 0x7f80u;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const bool inf = ((v >> (16 * h)) & kExp) == kExp && k + h >= node && k + h < end;
        bad |= inf;
        if (inf || k + h >= end) v &= h ? 0x0000ffffu : 0xffff0000u;
    }
    return v;
}

template <int D, bool FP8>
__global__ void __launch_bounds__(kThreads, 1) tree_few_kernel(const __grid_constant__ CUtensorMap tmk,
                                                               const __grid_constant__ CUtensorMap tmv,
                                                               const __grid_constant__ TreeArgs a) {
    using G_ = Geo<D, FP8>;
    constexpr int NS = G_::kStages;
    extern __shared__ uint8_t smem_raw[];
    __shared__ ShareScratch s_share;
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(sm + G_::kBarAt);
    uint64_t* empty = full + NS;
    uint64_t* pt_full = empty + NS;
    uint64_t* pt_empty = pt_full + kParts;
    uint64_t* x_in = pt_empty + kParts;  // every warp's share of a part is in shared memory
    uint64_t* x_out = x_in + 1;          // and has been read
    int* s_abort = reinterpret_cast<int*>(x_out + 1);
    int* s_bad = s_abort + 1;            // [2], by the part's parity: a drafted row's value is not finite
    Part* s_part = reinterpret_cast<Part*>(sm + G_::kPartAt);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < NS; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], kWarps / 2);
        }
        for (int s = 0; s < kParts; ++s) {
            mbar_init(&pt_full[s], 1);
            mbar_init(&pt_empty[s], kWarps);
        }
        mbar_init(x_in, kWarps);
        mbar_init(x_out, kWarps);
        *s_abort = 0;
        s_bad[0] = s_bad[1] = 0;
        s_share.pairs = 0;
        fence_barrier_init();
        prefetch_tensormap(&tmk);
        prefetch_tensormap(&tmv);
        work_at(a.work).join[blockIdx.x].parts = 0;
    }
    __syncthreads();
    using ItemWalk = Walk<kFewRows, kKeys>;
    const Share share = find_share<D, kThreads, ItemWalk>(a, s_share);
    const bool idle = share.lo >= share.hi;
    volatile int* abort_flag = s_abort;
    // A bounded wait.  After a time-out no role waits or loads any more, and
    // every role leaves at its next part.
    auto wait = [&](uint64_t* b, uint32_t parity) {
        if (mbar_try_wait(b, parity)) return;
        const uint64_t start = globaltimer_ns();
        while (!mbar_try_wait_sleep(b, parity, 100000u)) {
            if (*abort_flag) return;
            if (globaltimer_ns() - start > kWaitNs) *abort_flag = 1;
        }
    };

    if (idle) {
        // no share
    } else if (warp == kWarps) {
        // ------------------------------------------------ the walk and the loads
        ItemWalk w;
        w.start(a, share, s_share);
        const uint64_t policy = l2_evict_first();  // a key is read once
        int pos = 0;
        for (int idx = 0;; ++idx) {
            const int r = idx % kParts;
            if (idx >= kParts) wait(&pt_empty[r], ((idx / kParts) & 1u) ^ 1u);
            if (lane == 0) {
                s_part[r] = w.describe(a, share);
                mbar_arrive(&pt_full[r]);
            }
            __syncwarp();
            if (!w.valid || *abort_flag) break;
            if (lane == 0) {
                const int z = w.sq * a.nkv + w.g;
#pragma unroll 1
                for (int t = w.t0; t < w.t1; ++t, ++pos) {
                    const int s = pos % NS;
                    if (pos >= NS) wait(&empty[s], ((pos / NS) & 1u) ^ 1u);
                    if (*abort_flag) break;
                    uint8_t* dst = sm + s * 2 * G_::kTileBytes;
                    mbar_arrive_expect_tx(&full[s], 2 * G_::kTileBytes);
                    constexpr int kBoxes = FP8 ? 1 : D / 64;
#pragma unroll
                    for (int h = 0; h < kBoxes; ++h)
                        tma_load_3d_hint(dst + h * kKeys * 128, &tmk, &full[s], 64 * h, t * kKeys, z, policy);
#pragma unroll
                    for (int h = 0; h < kBoxes; ++h)
                        tma_load_3d_hint(dst + G_::kTileBytes + h * kKeys * 128, &tmv, &full[s], 64 * h, t * kKeys, z, policy);
                }
            }
            __syncwarp();
            w.seek(a, false);
        }
        if (lane == 0 && *abort_flag)  // the copies in flight land before the CTA leaves
            for (int j = max(0, pos - NS); j < pos; ++j) {
                const uint64_t t = globaltimer_ns();
                while (!mbar_try_wait(&full[j % NS], (j / NS) & 1u) && globaltimer_ns() - t < NF_WAIT_BUDGET_NS) {
                }
            }
    } else {
        // ------------------------------------------------ 16 keys of a tile
        const int grp = lane >> 2, t4 = lane & 3;  // fragment coordinates: rows grp and grp + 8
        const int mi = lane >> 3, mr = lane & 7;   // ldmatrix: the lane's matrix and row
        const int key0 = 16 * (warp & 3);          // the warp's keys of a tile
        float* s_out = reinterpret_cast<float*>(sm + G_::kOutAt);
        float2* s_ml = reinterpret_cast<float2*>(sm + G_::kMlAt);
        uint32_t pos0 = 0;  // tiles before the part
        for (int idx = 0;; ++idx) {
            wait(&pt_full[idx % kParts], (idx / kParts) & 1u);
            const Part& w = s_part[idx % kParts];
            if (*abort_flag || w.rows == 0) break;
            const int rows = w.rows, cnt = w.t1 - w.t0, first = w.first, p0 = w.p0, n = w.n;
            const bool two = rows > 8;
            const int t_first = w.t0 + static_cast<int>(((warp >> 2) ^ pos0) & 1u);  // this warp's tiles: every other one
            const int end = p0 + n;
            const int64_t zrow = static_cast<int64_t>(w.z) * a.L;
            // E4M3: lanes 0-15 hold the scales of the warp's 16 keys, lanes 16-31 the values' scales
            float sc = 0.f;
            auto fetch = [&](int t) {
                const int key = t * kKeys + key0 + (lane & 15);
                return key < end ? __ldg((lane < 16 ? a.k_scale : a.v_scale) + zrow + key) : 0.f;
            };
            if (FP8 && t_first < w.t1) sc = fetch(t_first);
            // q's fragments.  Step s of the product covers dims 16 s .. + 15; with E4M3 a thread's codes are four
            // neighbours, so its slots 2 t, 2 t + 1, 2 t + 8, 2 t + 9 stand for dims 4 t .. 4 t + 3.
            uint32_t qa[D / 16][4];
            int node[2];
            float cq[2] = {a.c, a.c};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = w.row0 + grp + 8 * h;
                node[h] = row / a.G;
                const bool in = grp + 8 * h < rows;
                const uint16_t* q = a.q + (static_cast<int64_t>(first + node[h]) * a.nq + w.g * a.G + (row - node[h] * a.G)) * D;
#pragma unroll
                for (int s = 0; s < D / 16; ++s) {
                    if (FP8) {
                        const uint2 v = in ? *reinterpret_cast<const uint2*>(q + 16 * s + 4 * t4) : make_uint2(0u, 0u);
                        qa[s][h] = v.x;
                        qa[s][2 + h] = v.y;
                    } else {
                        qa[s][h] = in ? *reinterpret_cast<const uint32_t*>(q + 16 * s + 2 * t4) : 0u;
                        qa[s][2 + h] = in ? *reinterpret_cast<const uint32_t*>(q + 16 * s + 2 * t4 + 8) : 0u;
                    }
                }
                if (FP8) {
                    // the row's largest exponent to 2^0: what F16 then loses is below 2^-24 of the row's maximum
                    uint32_t top = 0;
#pragma unroll
                    for (int s = 0; s < D / 16; ++s)
#pragma unroll
                        for (int e = 0; e < 4; e += 2) top = max(top, max(qa[s][h + e] & 0x7f80u, (qa[s][h + e] >> 16) & 0x7f80u));
                    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    const int e = top == 0 || top == 0x7f80u ? 127 : min(static_cast<int>(top >> 7), 253);
                    const float down = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
                    cq[h] = a.c * __uint_as_float(static_cast<uint32_t>(e) << 23);
#pragma unroll
                    for (int s = 0; s < D / 16; ++s)
#pragma unroll
                        for (int f = 0; f < 4; f += 2)
                            qa[s][h + f] = pack_f16x2(__uint_as_float(qa[s][h + f] << 16) * down,
                                                      __uint_as_float(qa[s][h + f] & 0xffff0000u) * down);
                }
            }
            float o[D / 8][4];
#pragma unroll
            for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
            float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
            // E4M3: the weights p * (value's scale) enter the product as F16 times inv, a power of two that keeps the
            // row's largest weight so far, ref (as the running max has it), within [2^-4, 2^15]
            float ref[2] = {0.f, 0.f}, inv[2] = {1.f, 1.f};
            bool bad = false;

#pragma unroll 1
            for (int t = t_first; t < w.t1; t += 2) {
                const uint32_t pos = pos0 + static_cast<uint32_t>(t - w.t0);
                const int s = static_cast<int>(pos % NS);
                const float my = sc;
                if (FP8 && t + 2 < w.t1) sc = fetch(t + 2);
                wait(&full[s], (pos / NS) & 1u);
                __syncwarp();
                const int k0 = t * kKeys + key0;  // the warp's first key
                if (k0 < end) {
                    const uint32_t kt = smem_u32(sm + s * 2 * G_::kTileBytes), vt = kt + G_::kTileBytes;
                    const bool tail = k0 + 16 > p0;
                    // ---- scores: n-tile j holds keys key0 + 8 j .. + 7
                    float x[2][4];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float even[4] = {0.f, 0.f, 0.f, 0.f}, odd[4] = {0.f, 0.f, 0.f, 0.f};
                        const int key = key0 + 8 * j + mr;
                        if (FP8) {
#pragma unroll
                            for (int c = 0; c < D / 16; c += 4) {
                                // 16-byte chunk c + mi of the key's row: a step's 16 codes
                                const uint32_t ch = c + mi;
                                uint32_t b[4];
                                ldsm_x4(kt + key * D + ((D == 128 ? ch ^ (key & 7) : ch ^ ((key >> 1) & 3)) << 4), b);
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    mma_f16(e & 1 ? odd : even, qa[c + e][0], qa[c + e][1], qa[c + e][2], qa[c + e][3],
                                            e4m3x2_to_f16x2(b[e]), e4m3x2_to_f16x2(b[e] >> 16));
                            }
                        } else {
#pragma unroll
                            for (int c = 0; c < D / 16; c += 2) {
                                const int dc = 16 * (c + (mi >> 1)) + 8 * (mi & 1);
                                uint32_t b[4];
                                ldsm_x4(kt + (dc >> 6) * kKeys * 128 + key * 128 + ((((dc & 63) >> 3) ^ (key & 7)) << 4), b);
                                mma_16816(even, qa[c][0], qa[c][1], qa[c][2], qa[c][3], b[0], b[1]);
                                mma_16816(odd, qa[c + 1][0], qa[c + 1][1], qa[c + 1][2], qa[c + 1][3], b[2], b[3]);
                            }
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[j][e] = even[e] + odd[e];
                    }
                    // ---- x = c q . k; the value e of n-tile j is row grp + 8 (e / 2), key 8 j + 2 t4 + (e & 1)
                    float vs[2][2];
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float ks = 1.f;
                            if (FP8) {
                                ks = __shfl_sync(0xffffffffu, my, 8 * j + 2 * t4 + e);
                                vs[j][e] = __shfl_sync(0xffffffffu, my, 16 + 8 * j + 2 * t4 + e);
                                if (tail && k0 + 8 * j + 2 * t4 + e >= p0 && !isfinite(vs[j][e])) {
                                    bad = true;
                                    vs[j][e] = 0.f;
                                }
                            }
                            x[j][e] *= ks * cq[0];
                            x[j][2 + e] *= ks * cq[1];
                        }
                    if (tail)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t vis = visible(a, first + node[h], node[h], n, k0 - p0, grp + 8 * h < rows);
#pragma unroll
                            for (int j = 0; j < 2; ++j)
#pragma unroll
                                for (int e = 0; e < 2; ++e)
                                    if (!((vis >> (8 * j + 2 * t4 + e)) & 1u)) x[j][2 * h + e] = -INFINITY;
                        }
                    // ---- the row's running maximum, sum and weights
                    uint32_t pa[4] = {0u, 0u, 0u, 0u};
                    float f[2] = {1.f, 1.f};
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (h == 1 && !two) break;
                        float mx = fmaxf(fmaxf(x[0][2 * h], x[0][2 * h + 1]), fmaxf(x[1][2 * h], x[1][2 * h + 1]));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                        const float mn = fmaxf(m[h], mx), mu = mn == -INFINITY ? 0.f : mn;
                        f[h] = m[h] == -INFINITY ? 0.f : ex2(m[h] - mu);
                        m[h] = mn;
                        float p[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) p[e] = ex2(x[e >> 1][2 * h + (e & 1)] - mu);
                        l[h] = l[h] * f[h] + ((p[0] + p[1]) + (p[2] + p[3]));
                        if (FP8) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) p[e] *= vs[e >> 1][e & 1];
                            float wm = fmaxf(fmaxf(fabsf(p[0]), fabsf(p[1])), fmaxf(fabsf(p[2]), fabsf(p[3])));
                            wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, 1));
                            wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, 2));
                            ref[h] = fmaxf(ref[h] * f[h], wm);
                            const float top = ref[h] * inv[h];
                            if (ref[h] > 0.f && !(top >= 0.0625f && top <= 32768.f)) {
                                const int e = min(max(258 - static_cast<int>(__float_as_uint(ref[h]) >> 23), 7), 247);
                                const float to = __uint_as_float(static_cast<uint32_t>(e) << 23);
                                f[h] *= fminf(to / inv[h], 1.7e38f);
                                inv[h] = to;
                            }
                            pa[h] = pack_f16x2(p[0] * inv[h], p[1] * inv[h]);
                            pa[2 + h] = pack_f16x2(p[2] * inv[h], p[3] * inv[h]);
                        } else {
                            pa[h] = pack_bf16x2(p[0], p[1]);
                            pa[2 + h] = pack_bf16x2(p[2], p[3]);
                        }
                    }
                    if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f)) {
#pragma unroll
                        for (int i = 0; i < D / 8; ++i) {
                            o[i][0] *= f[0];
                            o[i][1] *= f[0];
                            o[i][2] *= f[1];
                            o[i][3] *= f[1];
                        }
                    }
                    // ---- O += P V over the warp's 16 keys
                    const int vkey = key0 + 8 * (mi & 1) + mr, kk = k0 + 2 * t4;
                    if (FP8) {
#pragma unroll
                        for (int c = 0; c < D / 16; c += 2) {
                            // chunk c + mi / 2, keys 8 (mi & 1) .. + 7, pairs of codes transposed: a register holds dims
                            // 2 grp and 2 grp + 1 of keys 2 t4 and 2 t4 + 1
                            const uint32_t ch = c + (mi >> 1);
                            uint32_t b[4];
                            ldsm_x4_t(vt + vkey * D + ((D == 128 ? ch ^ (vkey & 7) : ch ^ ((vkey >> 1) & 3)) << 4), b);
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                const uint32_t lo = __byte_perm(b[2 * i], 0u, 0x3120), hi = __byte_perm(b[2 * i + 1], 0u, 0x3120);
#pragma unroll
                                for (int e = 0; e < 2; ++e) {  // dims 16 (c + i) + 2 (column) + e
                                    uint32_t b0 = e4m3x2_to_f16x2(e ? lo >> 16 : lo), b1 = e4m3x2_to_f16x2(e ? hi >> 16 : hi);
                                    if (tail) {
                                        b0 = clean<FP8>(b0, kk, p0, end, bad);
                                        b1 = clean<FP8>(b1, kk + 8, p0, end, bad);
                                    }
                                    mma_f16(o[2 * (c + i) + e], pa[0], pa[1], pa[2], pa[3], b0, b1);
                                }
                            }
                        }
                    } else {
#pragma unroll
                        for (int c = 0; c < D / 8; c += 2) {
                            const int dc = 8 * (c + (mi >> 1));
                            uint32_t b[4];
                            ldsm_x4_t(vt + (dc >> 6) * kKeys * 128 + vkey * 128 + ((((dc & 63) >> 3) ^ (vkey & 7)) << 4), b);
                            if (tail)
#pragma unroll
                                for (int e = 0; e < 4; ++e) b[e] = clean<FP8>(b[e], kk + 8 * (e & 1), p0, end, bad);
                            mma_16816(o[c], pa[0], pa[1], pa[2], pa[3], b[0], b[1]);
                            mma_16816(o[c + 1], pa[0], pa[1], pa[2], pa[3], b[2], b[3]);
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty[s]);
            }
            pos0 += static_cast<uint32_t>(cnt);
            // ---- the warps' outputs to shared memory
            if (bad) s_bad[idx & 1] = 1;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
                l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
                const int r = grp + 8 * h;
                if (r >= rows) continue;
                if (t4 == 0) s_ml[warp * kFewRows + r] = make_float2(m[h], l[h]);
                float* dst = s_out + (warp * kFewRows + r) * D;
                const float back = FP8 ? 1.f / inv[h] : 1.f;
                if (FP8) {
#pragma unroll
                    for (int c = 0; c < D / 16; ++c)
                        *reinterpret_cast<float4*>(dst + 16 * c + 4 * t4) =
                            make_float4(o[2 * c][2 * h] * back, o[2 * c + 1][2 * h] * back, o[2 * c][2 * h + 1] * back,
                                        o[2 * c + 1][2 * h + 1] * back);
                } else {
#pragma unroll
                    for (int c = 0; c < D / 8; ++c)
                        *reinterpret_cast<float2*>(dst + 8 * c + 2 * t4) = make_float2(o[c][2 * h], o[c][2 * h + 1]);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(x_in);
            wait(x_in, idx & 1u);
            // ---- and joined, four dims of a row a thread
            if (threadIdx.x == 0) s_bad[(idx + 1) & 1] = 0;
            const bool whole = w.kind == 3;
            const int slot = 2 * blockIdx.x + (w.kind & 1);
            const Work wk = work_at(a.work);
            for (int e = threadIdx.x; e < rows * (D / 4); e += 32 * kWarps) {
                const int r = e / (D / 4), d = e % (D / 4) * 4;
                float mt = -INFINITY, lt = 0.f;
#pragma unroll
                for (int k = 0; k < kWarps; ++k) mt = fmaxf(mt, s_ml[k * kFewRows + r].x);
                const float mu = mt == -INFINITY ? 0.f : mt;
                float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int k = 0; k < kWarps; ++k) {
                    const float2 v = s_ml[k * kFewRows + r];
                    const float4 x = *reinterpret_cast<const float4*>(s_out + (k * kFewRows + r) * D + d);
                    const float g = v.x == -INFINITY && v.y == 0.f ? 0.f : ex2(v.x - mu);
                    lt += v.y * g;
                    if (g != 0.f) {
                        acc.x = fmaf(x.x, g, acc.x);
                        acc.y = fmaf(x.y, g, acc.y);
                        acc.z = fmaf(x.z, g, acc.z);
                        acc.w = fmaf(x.w, g, acc.w);
                    }
                }
                const int row = w.row0 + r, nd = row / a.G;
                if (s_bad[idx & 1] && poisoned<D, FP8>(a, w.z, p0, n, first, nd)) lt = NAN;
                if (whole) {
                    const float iv = lt == 0.f ? 0.f : 1.f / lt;
                    uint16_t* dst = a.out + (static_cast<int64_t>(first + nd) * a.nq + w.g * a.G + (row - nd * a.G)) * D + d;
                    *reinterpret_cast<uint2*>(dst) = make_uint2(bf16x2_hw(acc.x * iv, acc.y * iv), bf16x2_hw(acc.z * iv, acc.w * iv));
                } else {
                    const int64_t at = static_cast<int64_t>(slot) * kItemRows + r;
                    *reinterpret_cast<float4*>(wk.acc + at * D + d) = acc;
                    if (d == 0) wk.ml[at] = make_float2(mu, lt);
                }
            }
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(x_out);
                mbar_arrive(&pt_empty[idx % kParts]);
            }
            wait(x_out, idx & 1u);
        }
    }
    __syncwarp();
    pdl_trigger();
    __syncthreads();
    if (threadIdx.x == 0 && *abort_flag && a.status) atomicCAS(a.status, 0, NF_DEVERR_WAIT_FULL);
}

template <int D, bool FP8>
cudaError_t launch(const nf_kv_cache& c, const TreeArgs& a, int grid, cudaStream_t st) {
    CUtensorMap tmk, tmv;
    const uint64_t heads = static_cast<uint64_t>(c.seqs) * c.kv_heads;
    if (!make_tmap_kv(&tmk, c.k, !FP8, D, c.max_context, heads, kKeys, true) ||
        !make_tmap_kv(&tmv, c.v, !FP8, D, c.max_context, heads, kKeys, true))
        return cudaErrorInvalidValue;
    static bool attr[kMaxDevices] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
    constexpr int smem = Geo<D, FP8>::kSmem;
    if (!attr[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(tree_few_kernel<D, FP8>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        attr[dev] = true;
    }
    tree_few_kernel<D, FP8><<<grid, kThreads, smem, st>>>(tmk, tmv, a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_tree_few(const nf_kv_cache& c, const TreeArgs& a, int grid, cudaStream_t st) {
    const bool fp8 = c.kind == NF_KV_E4M3;
    if (c.head_dim == 128) return fp8 ? launch<128, true>(c, a, grid, st) : launch<128, false>(c, a, grid, st);
    return fp8 ? launch<64, true>(c, a, grid, st) : launch<64, false>(c, a, grid, st);
}

}  // namespace nf
