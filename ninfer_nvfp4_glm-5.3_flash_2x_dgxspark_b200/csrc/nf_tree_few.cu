// nf_tree_few.cu -- nf_tree_attention's kernel for few rows of a sequence and
// KV head (decode, and trees of a node or two): warp-level tensor-core tiles.
//
// The work is the cache's bytes: 8 rows do 8 (BF16) or 16 (E4M3) flops a
// byte (a row 4 D flops on a key of 4 D or 2 D bytes), a fraction of what the tensor cores could.  So the keys only have to
// stream: one warp issues TMA tiles of 64 keys into a ring, and eight warps
// take 32 keys of a tile each (pairs of warps take tiles in turn), with their
// own running maximum, sum and output in registers.  Two more warps bring the
// next part's q into fragments' order and join the eight warps' outputs of the
// part before, so that the others go from part to part without a stop.  Both
// products are taken transposed, S^T = K Q^T and O^T = V^T P^T, so that the keys and the head's dims fill the 16 rows of the m16n8k16
// tiles and the 8 columns are the rows of q.  E4M3 codes become F16 in
// registers, one conversion for two codes and nothing written back to shared
// memory; q's rows are brought into F16's range by a power of two, and so are
// the probabilities times the values' scales (see `ref` below).
//
// What bounds it: with many keys the instructions of a tile and their fetch
// (the hot loop fits the instruction cache since the rare paths left it: 137 to
// 88 us), then the bytes.  256 sequences of one row, 8 rows a KV head, on up to
// 2,048 E4M3 keys: 82 to 85 us, 5.0 TB/s; one such row on 1,000 keys: 14 us, of
// which 8 the kernel's own latency and 3 the join's launch.
#include "nf_tree.cuh"

#include <cmath>

namespace nf {

namespace {

constexpr int kKeys = 64;     // keys per tile

// NT: column tiles of 8 rows (1, or with BF16 2).
template <int D, bool FP8, int NT>
struct Geo {
    static constexpr int kWarps = 8;            // consuming warps
    static constexpr int kGroups = kWarps / 2;  // which take tiles in turn
    static constexpr int kAux = 2;              // warps for q and the join
    static constexpr int kThreads = 32 * (kWarps + 1 + kAux);
    static constexpr int kRows = 8 * NT;
    static constexpr int kPitch = D + 8;        // floats of an output row in shared memory
    static constexpr int kTileBytes = kKeys * D * (FP8 ? 1 : 2);  // K or V
    // A multiple of kGroups: then a stage is always the same group's, which has waited for its load before when it waits
    // for the next.  Loads may land out of order, and another group's wait could take the phase before for its own.
    static constexpr int kStages = FP8 ? 8 : 4;
    static_assert(kStages % kGroups == 0);
    static constexpr int kOutAt = kStages * 2 * kTileBytes;             // [warp][row][D] floats
    static constexpr int kMlAt = kOutAt + kWarps * kRows * kPitch * 4;  // [warp][row] (m, l)
    static constexpr int kQPitch = 2 * D + 16;  // bytes of a row of q
    static constexpr int kQAt = kMlAt + kWarps * kRows * 8;             // [2][row] q as F16 or BF16
    static constexpr int kCqAt = kQAt + 2 * kRows * kQPitch;            // [2][row] factors
    static constexpr int kPartAt = kCqAt + 2 * kRows * 4;
    static constexpr int kBarAt = kPartAt + kParts * static_cast<int>(sizeof(Part));
    static constexpr int kSmem = 1024 + kBarAt + (2 * kStages + 2 * kParts + 6) * 8 + 32;
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
// An 8 x 8 matrix of 16-bit values held as fragments, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

template <int D, bool FP8, int NT>
__global__ void __launch_bounds__(Geo<D, FP8, NT>::kThreads, 1) tree_few_kernel(const __grid_constant__ CUtensorMap tmk,
                                                               const __grid_constant__ CUtensorMap tmv,
                                                               const __grid_constant__ TreeArgs a) {
    using G_ = Geo<D, FP8, NT>;
    constexpr int NS = G_::kStages, kWarps = G_::kWarps, kRows = G_::kRows, kPitch = G_::kPitch;
    extern __shared__ uint8_t smem_raw[];
    __shared__ ShareScratch s_share;
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(sm + G_::kBarAt);
    uint64_t* empty = full + NS;
    uint64_t* pt_full = empty + NS;
    uint64_t* pt_empty = pt_full + kParts;
    uint64_t* x_in = pt_empty + kParts;  // every warp's share of a part is in shared memory
    uint64_t* x_out = x_in + 1;          // and has been read
    uint64_t* q_full = x_out + 1;        // [2] a part's q
    uint64_t* q_empty = q_full + 2;
    int* s_abort = reinterpret_cast<int*>(q_empty + 2);
    int* s_bad = s_abort + 1;            // [4], of the part in turn: a drafted row's value is not finite
    Part* s_part = reinterpret_cast<Part*>(sm + G_::kPartAt);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < NS; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 2);
        }
        for (int s = 0; s < kParts; ++s) {
            mbar_init(&pt_full[s], 1);
            mbar_init(&pt_empty[s], kWarps + G_::kAux);
        }
        mbar_init(x_in, kWarps);
        mbar_init(x_out, G_::kAux);
        for (int s = 0; s < 2; ++s) {
            mbar_init(&q_full[s], G_::kAux);
            mbar_init(&q_empty[s], kWarps);
        }
        *s_abort = 0;
        for (int s = 0; s < 4; ++s) s_bad[s] = 0;
        fence_barrier_init();
        prefetch_tensormap(&tmk);
        prefetch_tensormap(&tmv);
        work_at(a.work).join[blockIdx.x].parts = 0;
        work_at(a.work).marks[blockIdx.x] = 0;
    }
    __syncthreads();
    pdl_trigger();  // the join's blocks may wait for this grid beside it
    // an item's start and end take the time of about eight tiles (E4M3, D 128): 83 us above, without that weight 90
    using ItemWalk = Walk<kRows, kKeys, 8, 1, 1>;
    const Share share = find_share<D, G_::kThreads, G_::kGroups, ItemWalk>(a, s_share);
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
    } else if (warp > kWarps) {
        // ------------------------------------------------ q, and the join
        const int tid = threadIdx.x - 32 * (kWarps + 1);
        constexpr int kCount = 32 * G_::kAux, C = D / 8;  // 16-byte chunks of a row of q
        const float* s_out = reinterpret_cast<const float*>(sm + G_::kOutAt);
        const float2* s_ml = reinterpret_cast<const float2*>(sm + G_::kMlAt);
#pragma unroll 1
        for (int idx = 0;; ++idx) {
            wait(&pt_full[idx % kParts], (idx / kParts) & 1u);
            const bool more = !*abort_flag && s_part[idx % kParts].rows > 0;
            if (more) {
                const Part& w = s_part[idx % kParts];
                const int b = idx & 1;
                if (idx >= 2) wait(&q_empty[b], ((idx >> 1) & 1u) ^ 1u);
#pragma unroll
                for (int e = tid; e < kRows * C; e += kCount) {
                    const int r = e / C, ch = e % C, row = w.row0 + r, node = row / a.G;
                    uint4 v = make_uint4(0u, 0u, 0u, 0u);
                    if (r < w.rows)
                        v = *reinterpret_cast<const uint4*>(
                            a.q + (static_cast<int64_t>(w.first + node) * a.nq + w.g * a.G + (row - node * a.G)) * D + 8 * ch);
                    float mine = a.c;
                    if (FP8) {
                        // the row's largest exponent to 2^0: what F16 then loses is below 2^-24 of the row's maximum
                        uint32_t in[4] = {v.x, v.y, v.z, v.w}, top = 0;
#pragma unroll
                        for (int k = 0; k < 4; ++k) top = max(top, max(in[k] & 0x7f80u, (in[k] >> 16) & 0x7f80u));
#pragma unroll
                        for (int o = 1; o < C; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
                        const int ex = top == 0 || top == 0x7f80u ? 127 : min(static_cast<int>(top >> 7), 253);
                        const float down = __uint_as_float(static_cast<uint32_t>(254 - ex) << 23);
                        mine = a.c * __uint_as_float(static_cast<uint32_t>(ex) << 23);
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            in[k] = pack_f16x2(__uint_as_float(in[k] << 16) * down, __uint_as_float(in[k] & 0xffff0000u) * down);
                        v = make_uint4(in[0], in[1], in[2], in[3]);
                    }
                    *reinterpret_cast<uint4*>(sm + G_::kQAt + (b * kRows + r) * G_::kQPitch + 16 * ch) = v;
                    if (ch == 0) reinterpret_cast<float*>(sm + G_::kCqAt)[b * kRows + r] = mine;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_full[b]);
            }
            if (idx > 0) {
                // the part before: four dims of a row a thread
                const int at = idx - 1;
                const Part& w = s_part[at % kParts];
                wait(x_in, at & 1u);
                if (tid == 0) s_bad[(at + 2) & 3] = 0;
                const int rows = w.rows;
                const bool whole = w.kind == 3;
                const int slot = 2 * blockIdx.x + (w.kind & 1);
                const Work wk = work_at(a.work);
                uint32_t nan_rows = 0;
                if (__any_sync(0xffffffffu, s_bad[at & 3] != 0)) {  // a lane a row
                    const int node = (w.row0 + min(lane, rows - 1)) / a.G;
                    nan_rows = __ballot_sync(0xffffffffu, poisoned<D, FP8>(a, w.z, w.p0, w.n, w.first, node, lane < rows));
                }
#pragma unroll 1
                for (int e = tid; e < rows * (D / 4); e += kCount) {
                    const int r = e / (D / 4), d = e % (D / 4) * 4;
                    float2 ml[kWarps];
                    float mt = -INFINITY, lt = 0.f;
#pragma unroll
                    for (int k = 0; k < kWarps; ++k) {
                        ml[k] = s_ml[k * kRows + r];
                        mt = fmaxf(mt, ml[k].x);
                    }
                    const float mu = mt == -INFINITY ? 0.f : mt;
                    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int k = 0; k < kWarps; ++k) {
                        const float4 x = *reinterpret_cast<const float4*>(s_out + (k * kRows + r) * kPitch + d);
                        const float g = ml[k].x == -INFINITY && ml[k].y == 0.f ? 0.f : ex2(ml[k].x - mu);
                        lt += ml[k].y * g;
                        acc.x += g == 0.f ? 0.f : x.x * g;
                        acc.y += g == 0.f ? 0.f : x.y * g;
                        acc.z += g == 0.f ? 0.f : x.z * g;
                        acc.w += g == 0.f ? 0.f : x.w * g;
                    }
                    const int row = w.row0 + r, nd = row / a.G;
                    if ((nan_rows >> r) & 1u) lt = NAN;
                    if (whole) {
                        const float iv = lt == 0.f ? 0.f : 1.f / lt;
                        uint16_t* dst = a.out + (static_cast<int64_t>(w.first + nd) * a.nq + w.g * a.G + (row - nd * a.G)) * D + d;
                        *reinterpret_cast<uint2*>(dst) =
                            make_uint2(bf16x2_hw(acc.x * iv, acc.y * iv), bf16x2_hw(acc.z * iv, acc.w * iv));
                    } else {
                        const int64_t to = static_cast<int64_t>(slot) * kItemRows + r;
                        *reinterpret_cast<float4*>(wk.acc + to * D + d) = acc;
                        if (d == 0) wk.ml[to] = make_float2(mu, lt);
                    }
                }
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(x_out);
                    mbar_arrive(&pt_empty[at % kParts]);
                }
            }
            if (!more) break;
        }
    } else {
        // ------------------------------------------------ 32 keys of a tile
        // Fragment coordinates: of S^T and O^T a thread holds rows 2 t4, 2 t4 + 1 of a column tile for keys (dims)
        // grp and grp + 8.
        const int grp = lane >> 2, t4 = lane & 3;
        const int mi = lane >> 3, mr = lane & 7;  // ldmatrix: the lane's matrix and row
        const int key0 = 32 * (warp & 1);         // the warp's keys of a tile
        float* s_out = reinterpret_cast<float*>(sm + G_::kOutAt);
        float2* s_ml = reinterpret_cast<float2*>(sm + G_::kMlAt);
        uint32_t pos0 = 0;  // tiles before the part
        wait(&pt_full[0], 0);
        // E4M3: the scales of the warp's next 32 keys, one a lane
        float ksc = 0.f, vsc = 0.f;
        auto fetch = [&](const Part& w, int t) {
            const int key = t * kKeys + key0 + lane;
            const bool in = t < w.t1 && key < w.p0 + w.n;
            const int64_t at = static_cast<int64_t>(w.z) * a.L + key;
            ksc = in ? __ldg(a.k_scale + at) : 0.f;
            vsc = in ? __ldg(a.v_scale + at) : 0.f;
        };
        // a part's first tile of this warp: every kGroups-th in the order of all tiles
        auto first_tile = [&](const Part& w) { return w.t0 + static_cast<int>(((warp >> 1) - pos0) % G_::kGroups); };
        if (FP8 && !*abort_flag) fetch(s_part[0], first_tile(s_part[0]));
#pragma unroll 1
        for (int idx = 0;; ++idx) {
            const Part& w = s_part[idx % kParts];
            if (*abort_flag || w.rows == 0) break;
            const int rows = w.rows, t1 = w.t1, first = w.first, p0 = w.p0, n = w.n, end = p0 + n;
            const int t_first = first_tile(w);
            // q's fragments, row 8 c + grp of column tile c.  Step s of the product covers dims 16 s .. + 15; with E4M3
            // a thread's codes are four neighbours, so its slots 2 t, 2 t + 1, 2 t + 8, 2 t + 9 stand for dims 4 t .. + 3.
            uint32_t qb[NT][D / 16][2];
            float cq[NT][2];
            wait(&q_full[idx & 1], (idx >> 1) & 1u);
            __syncwarp();
#pragma unroll
            for (int c = 0; c < NT; ++c) {
                const uint8_t* q = sm + G_::kQAt + ((idx & 1) * kRows + 8 * c + grp) * G_::kQPitch;
#pragma unroll
                for (int s = 0; s < D / 16; ++s) {
                    if (FP8) {
                        const uint2 v = *reinterpret_cast<const uint2*>(q + 32 * s + 8 * t4);
                        qb[c][s][0] = v.x;
                        qb[c][s][1] = v.y;
                    } else {
                        qb[c][s][0] = *reinterpret_cast<const uint32_t*>(q + 32 * s + 4 * t4);
                        qb[c][s][1] = *reinterpret_cast<const uint32_t*>(q + 32 * s + 4 * t4 + 16);
                    }
                }
                const float2 f = *reinterpret_cast<const float2*>(sm + G_::kCqAt + ((idx & 1) * kRows + 8 * c + 2 * t4) * 4);
                cq[c][0] = f.x;
                cq[c][1] = f.y;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_empty[idx & 1]);
            float o[NT][D / 16][4];
#pragma unroll
            for (int c = 0; c < NT; ++c)
#pragma unroll
                for (int i = 0; i < D / 16; ++i) o[c][i][0] = o[c][i][1] = o[c][i][2] = o[c][i][3] = 0.f;
            // E4M3: the weights p * (value's scale) enter the product as F16 times inv, a power of two that keeps the
            // row's largest weight so far, ref (as the running max has it), within [2^8, 2^15]: F16's last place is then
            // below 2^-32 of it, where a weight is rounded otherwise by 2^-11 of itself
            float m[NT][2], l[NT][2], ref[NT][2], inv[NT][2];
#pragma unroll
            for (int c = 0; c < NT; ++c)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    m[c][e] = -INFINITY;
                    l[c][e] = ref[c][e] = 0.f;
                    inv[c][e] = 1.f;
                }
            bool bad = false;

#pragma unroll 1
            for (int t = t_first; t < t1; t += G_::kGroups) {
                const uint32_t pos = pos0 + static_cast<uint32_t>(t - w.t0);
                const int s = static_cast<int>(pos % NS);
                const float my_k = ksc, my_v = vsc;
                if (FP8) fetch(w, t + G_::kGroups);
                wait(&full[s], (pos / NS) & 1u);
                __syncwarp();
                const int k0 = t * kKeys + key0;  // the warp's first key
                if (k0 < end) {
                    const uint32_t kt = smem_u32(sm + s * 2 * G_::kTileBytes), vt = kt + G_::kTileBytes;
                    const bool tail = k0 + 32 > p0;
                    if (__builtin_expect(tail, 0)) {
                        // V's rows behind the sequence, and drafted rows that are not finite (which is noted), become
                        // zeros: a zero probability must not meet a NaN.  A lane has a key's row.
                        const int row = key0 + lane, at = k0 + lane;
                        uint8_t* v = sm + s * 2 * G_::kTileBytes + G_::kTileBytes;
                        constexpr int kRowBytes = D * (FP8 ? 1 : 2), kBox = FP8 ? kRowBytes : 128;
                        bool zero = at >= end;
                        if (at >= p0 && at < end)
#pragma unroll 1
                            for (int c = 0; c < kRowBytes / 16; ++c) {  // chunks in any order: the swizzle stays in the row
                                const uint4 x = *reinterpret_cast<const uint4*>(v + c * 16 / kBox * (kKeys * kBox) + row * kBox + c * 16 % kBox);
                                const uint32_t in[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                                for (int k = 0; k < 4; ++k)  // an exponent of all ones (E4M3: 0x7f) carries into the sign's place
                                    zero |= FP8 ? (((in[k] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0
                                                : (((in[k] & 0x7f807f80u) + 0x00800080u) & 0x80008000u) != 0;
                            }
                        if (zero) {
                            bad |= at < end;
#pragma unroll 1
                            for (int c = 0; c < kRowBytes / 16; ++c)
                                *reinterpret_cast<uint4*>(v + c * 16 / kBox * (kKeys * kBox) + row * kBox + c * 16 % kBox) = make_uint4(0u, 0u, 0u, 0u);
                        }
                        fence_proxy_async();  // before TMA writes here again
                        __syncwarp();
                    }
                    // ---- S^T of 16 keys (b), twice
                    float x[NT][2][4];
#pragma unroll
                    for (int c = 0; c < NT; ++c)
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[c][0][e] = x[c][1][e] = 0.f;
#pragma unroll
                    for (int i = 0; i < D / 16; i += FP8 ? 2 : 1)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int key = key0 + 16 * h + 8 * (mi & 1) + mr;
                            uint32_t b[4];
                            if (FP8) {
                                // 16-byte chunks i and i + 1 (a step's 16 codes) of keys 0-7 and 8-15
                                const uint32_t ch = i + (mi >> 1);
                                ldsm_x4(kt + key * D + ((D == 128 ? ch ^ (key & 7) : ch ^ ((key >> 1) & 3)) << 4), b);
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const uint32_t a0 = e4m3x2_to_f16x2(b[2 * e]), a2 = e4m3x2_to_f16x2(b[2 * e] >> 16);
                                    const uint32_t a1 = e4m3x2_to_f16x2(b[2 * e + 1]), a3 = e4m3x2_to_f16x2(b[2 * e + 1] >> 16);
#pragma unroll
                                    for (int c = 0; c < NT; ++c) mma_f16(x[c][h], a0, a1, a2, a3, qb[c][i + e][0], qb[c][i + e][1]);
                                }
                            } else {
                                const int ch = 2 * i + (mi >> 1);
                                ldsm_x4(kt + (ch >> 3) * kKeys * 128 + key * 128 + (((ch & 7) ^ (key & 7)) << 4), b);
#pragma unroll
                                for (int c = 0; c < NT; ++c) mma_16816(x[c][h], b[0], b[1], b[2], b[3], qb[c][i][0], qb[c][i][1]);
                            }
                        }
                    // ---- x = c q . k; element (h, e): key 16 h + grp + 8 (e / 2), row 2 t4 + (e & 1)
                    float ks[4] = {1.f, 1.f, 1.f, 1.f}, vs[4] = {1.f, 1.f, 1.f, 1.f};
                    if (FP8)
#pragma unroll
                        for (int h = 0; h < 4; ++h) {
                            ks[h] = __shfl_sync(0xffffffffu, my_k, grp + 8 * h);
                            vs[h] = __shfl_sync(0xffffffffu, my_v, grp + 8 * h);
                            if (tail && k0 + grp + 8 * h >= p0 && !isfinite(vs[h])) {
                                bad = true;
                                vs[h] = 0.f;
                            }
                        }
                    uint32_t pb[NT][4];
                    bool scale = false;
                    float f[NT][2];
#pragma unroll
                    for (int c = 0; c < NT; ++c) {
                        float p[4][2];  // [key grp + 8 h][row]
#pragma unroll
                        for (int h = 0; h < 4; ++h)
#pragma unroll
                            for (int e = 0; e < 2; ++e) p[h][e] = x[c][h >> 1][2 * (h & 1) + e] * (ks[h] * cq[c][e]);
                        if (__builtin_expect(tail, 0))
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const int r = 8 * c + 2 * t4 + e, node = (w.row0 + r) / a.G;
                                const uint32_t vis = visible(a, first + node, node, n, k0 - p0, r < rows) >> grp;
#pragma unroll
                                for (int h = 0; h < 4; ++h)
                                    if (!((vis >> (8 * h)) & 1u)) p[h][e] = -INFINITY;
                            }
                        // ---- the rows' running maximum, sum and weights
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float mx = fmaxf(fmaxf(p[0][e], p[1][e]), fmaxf(p[2][e], p[3][e]));
                            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                            const float mn = fmaxf(m[c][e], mx), mu = mn == -INFINITY ? 0.f : mn;
                            f[c][e] = m[c][e] == -INFINITY ? 0.f : ex2(m[c][e] - mu);
                            m[c][e] = mn;
#pragma unroll
                            for (int h = 0; h < 4; ++h) p[h][e] = ex2(p[h][e] - mu);
                            l[c][e] = l[c][e] * f[c][e] + ((p[0][e] + p[1][e]) + (p[2][e] + p[3][e]));
                            if (FP8) {
#pragma unroll
                                for (int h = 0; h < 4; ++h) p[h][e] *= vs[h];
                                float wm = fmaxf(fmaxf(fabsf(p[0][e]), fabsf(p[1][e])), fmaxf(fabsf(p[2][e]), fabsf(p[3][e])));
                                wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, 4));
                                wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, 8));
                                wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, 16));
                                ref[c][e] = fmaxf(ref[c][e] * f[c][e], wm);
                                const float top = ref[c][e] * inv[c][e];
                                if (__builtin_expect(ref[c][e] > 0.f && !(top >= 256.f && top <= 32768.f), 0)) {
                                    const int ex = min(max(266 - static_cast<int>(__float_as_uint(ref[c][e]) >> 23), 7), 247);
                                    const float to = __uint_as_float(static_cast<uint32_t>(ex) << 23);
                                    f[c][e] *= fminf(to / inv[c][e], 1.7e38f);
                                    inv[c][e] = to;
                                }
#pragma unroll
                                for (int h = 0; h < 4; ++h) p[h][e] *= inv[c][e];
                            }
                            scale |= f[c][e] != 1.f;
                        }
#pragma unroll
                        for (int h = 0; h < 4; ++h)
                            pb[c][h] = transpose8(FP8 ? pack_f16x2(p[h][0], p[h][1]) : pack_bf16x2(p[h][0], p[h][1]));
                    }
                    if (__builtin_expect(__any_sync(0xffffffffu, scale), 0))
#pragma unroll
                        for (int c = 0; c < NT; ++c)
#pragma unroll
                            for (int i = 0; i < D / 16; ++i)
#pragma unroll
                                for (int e = 0; e < 4; ++e) o[c][i][e] *= f[c][e & 1];
                    // ---- O^T += V^T P^T over the warp's keys
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
#pragma unroll
                        for (int i = 0; i < D / 16; i += FP8 ? 2 : 1) {
                            uint32_t b[4];
                            if (FP8) {
                                // chunks i and i + 1 of keys 0-7 and 8-15, pairs of codes transposed: a register holds
                                // dims 2 grp and 2 grp + 1 (the tile's rows grp and grp + 8) of keys 2 t4 and 2 t4 + 1
                                const uint32_t ch = i + (mi >> 1);
                                const int key = key0 + 16 * h + 8 * (mi & 1) + mr;
                                ldsm_x4_t(vt + key * D + ((D == 128 ? ch ^ (key & 7) : ch ^ ((key >> 1) & 3)) << 4), b);
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const uint32_t lo = __byte_perm(b[2 * e], 0u, 0x3120), hi = __byte_perm(b[2 * e + 1], 0u, 0x3120);
                                    const uint32_t v[4] = {e4m3x2_to_f16x2(lo), e4m3x2_to_f16x2(lo >> 16), e4m3x2_to_f16x2(hi),
                                                           e4m3x2_to_f16x2(hi >> 16)};
#pragma unroll
                                    for (int c = 0; c < NT; ++c)
                                        mma_f16(o[c][i + e], v[0], v[1], v[2], v[3], pb[c][2 * h], pb[c][2 * h + 1]);
                                }
                            } else {
                                const int key = key0 + 16 * h + 8 * (mi >> 1) + mr, ch = 2 * i + (mi & 1);
                                ldsm_x4_t(vt + (ch >> 3) * kKeys * 128 + key * 128 + (((ch & 7) ^ (key & 7)) << 4), b);
#pragma unroll
                                for (int c = 0; c < NT; ++c)
                                    mma_16816(o[c][i], b[0], b[1], b[2], b[3], pb[c][2 * h], pb[c][2 * h + 1]);
                            }
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty[s]);
            }
            pos0 += static_cast<uint32_t>(t1 - w.t0);
            {
                // the next part's first scales are on their way meanwhile
                const int r = (idx + 1) % kParts;
                wait(&pt_full[r], ((idx + 1) / kParts) & 1u);
                if (FP8 && !*abort_flag) fetch(s_part[r], first_tile(s_part[r]));
            }
            // ---- the warp's output to shared memory, once the part before's has been read
            if (bad) s_bad[idx & 3] = 1;
            if (idx > 0) wait(x_out, (idx - 1) & 1u);
            __syncwarp();
#pragma unroll
            for (int c = 0; c < NT; ++c)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float lt = l[c][e];
                    lt += __shfl_xor_sync(0xffffffffu, lt, 4);
                    lt += __shfl_xor_sync(0xffffffffu, lt, 8);
                    lt += __shfl_xor_sync(0xffffffffu, lt, 16);
                    const int r = 8 * c + 2 * t4 + e;
                    if (r >= rows) continue;
                    if (grp == 0) s_ml[warp * kRows + r] = make_float2(m[c][e], lt);
                    float* dst = s_out + (warp * kRows + r) * kPitch;
                    const float back = FP8 ? 1.f / inv[c][e] : 1.f;
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                        if (FP8) {
                            *reinterpret_cast<float2*>(dst + 16 * i + 2 * grp) = make_float2(o[c][i][e] * back, o[c][i][2 + e] * back);
                        } else {
                            dst[16 * i + grp] = o[c][i][e];
                            dst[16 * i + 8 + grp] = o[c][i][2 + e];
                        }
                    }
                }
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(x_in);
                mbar_arrive(&pt_empty[idx % kParts]);
            }
        }
    }
    __syncthreads();
    if (threadIdx.x == 0 && *abort_flag) {
        work_at(a.work).marks[blockIdx.x] = kMarkGaveUp;
        if (a.status) atomicCAS(a.status, 0, NF_DEVERR_WAIT_FULL);
    }
}

template <int D, bool FP8, int NT>
cudaError_t launch(const nf_kv_cache& c, const TreeArgs& a, int grid, cudaStream_t st) {
    CUtensorMap tmk, tmv;
    const uint64_t heads = static_cast<uint64_t>(c.seqs) * c.kv_heads;
    if (!make_tmap_kv(&tmk, c.k, !FP8, D, c.max_context, heads, kKeys, true) ||
        !make_tmap_kv(&tmv, c.v, !FP8, D, c.max_context, heads, kKeys, true))
        return cudaErrorInvalidValue;
    static bool attr[kMaxDevices] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
    using G_ = Geo<D, FP8, NT>;
    if (!attr[dev]) {
        const cudaError_t e =
            cudaFuncSetAttribute(tree_few_kernel<D, FP8, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, G_::kSmem);
        if (e != cudaSuccess) return e;
        attr[dev] = true;
    }
    tree_few_kernel<D, FP8, NT><<<grid, G_::kThreads, G_::kSmem, st>>>(tmk, tmv, a);
    return cudaGetLastError();
}
template <int D>
cudaError_t launch_dim(const nf_kv_cache& c, const TreeArgs& a, int nt, int grid, cudaStream_t st) {
    return c.kind == NF_KV_E4M3 ? launch<D, true, 1>(c, a, grid, st)
           : nt == 1            ? launch<D, false, 1>(c, a, grid, st)
                                : launch<D, false, 2>(c, a, grid, st);
}

}  // namespace

cudaError_t launch_tree_few(const nf_kv_cache& c, const TreeArgs& a, int nt, int grid, cudaStream_t st) {
    return c.head_dim == 128 ? launch_dim<128>(c, a, nt, grid, st) : launch_dim<64>(c, a, nt, grid, st);
}

}  // namespace nf
