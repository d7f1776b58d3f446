// nf_tree.cu -- nf_tree_attention (include/nf_moe.h): attention of a
// sequence's new rows, one token, a chain or a tree, over its cached prefix
// and over one another.
//
// The kernel for many rows.  A tile of 128 keys is multiplied with 128 rows on
// the 5th-generation tensor cores, scores and outputs in TMEM, in two streams
// that take turns: while one stream's scores go through the softmax, the other
// stream's products run.  An item of more than 128 rows gives each stream its
// own 128 rows over the same tiles; a smaller one gives them every other tile.
//
// Per tile of 128 keys and 256 rows (D 128) the tensor cores need 2,048 cycles
// and the exponentials 2,048; it takes 6,000.  What bounds it is the chain of a
// stream: scores (512 cycles), softmax (about 3,000 beside the other stream's
// and the E4M3 widening on the same schedulers), product with V (512), and the
// barriers between them; a stream's scores and probabilities
// share their 128 TMEM columns, as two streams with outputs of 128 columns
// leave no room for a second set.  More and smaller tasks (64 keys, scores a
// task ahead) took 20% longer, twice the softmax warps 8%.
// The softmax subtracts the maxima that the tiles before had: no weight gets
// beyond 2^8 with them, or they rise (227 to 223 us).
// 4 sequences of 64 nodes, 8 rows a node, on up to 65,000 E4M3 keys: 224 us,
// 588 TFLOP/s; 24 of 16 nodes on 8,191 BF16 keys, where a tile of 128 rows
// waits for its 64 KB more than for the products: 76 to 84 us from run to run,
// 3.6 to 4.0 TB/s.
#include "nf_tree.cuh"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace nf {

namespace {

constexpr int kKeys = 128;       // keys per tile
constexpr int kThreads = 512;
constexpr int kConvWarp = 8, kTmaWarp = 12, kMmaWarp = 13, kRowWarp = 14, kScaleWarp = 15;
constexpr int kBadRing = 16;
constexpr float kRescale = 8.f;  // the running max may lag the true one by 2^8

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
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ void f16x2_to_f32(uint32_t v, float& lo, float& hi) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}"
        : "=f"(lo), "=f"(hi)
        : "r"(v));
}
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xffffffff;\n\tselp.u32 %0, 1, 0, P;\n\t}" : "=r"(p));
    return p;
}
// 32 lanes x 32 consecutive 32-bit columns
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
                 "%13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, "
                 "%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
                   "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
                   "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
                   "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr)
                 : "memory");
}

  // 16 lanes x 128 columns as matrix fragments: thread t holds columns 8 i + 2 (t % 4) and + 1 of lane t / 4 in r[4 i] and
// r[4 i + 1], and of lane t / 4 + 8 in r[4 i + 2] and r[4 i + 3].
__device__ __forceinline__ void tmem_ld_frag(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
                 "%13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
                 "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, "
                 "%51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
                   "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
                   "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
                   "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]),
                   "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]),
                   "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]),
                   "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]),
                   "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
                 : "r"(taddr)
                 : "memory");
}
// The same of 16 columns.
__device__ __forceinline__ void tmem_ld_frag16(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_st_frag16(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.16x256b.x2.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
// 16 lanes x 64 columns: thread t's column 4 i + t % 4 of lane t / 4 in r[2 i], of lane t / 4 + 8 in r[2 i + 1].
__device__ __forceinline__ void tmem_st_pairs(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.16x128b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
                 "%12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, "
                 "%31, %32};" ::"r"(taddr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
                   "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
                   "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
                   "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// D[tmem] (+)= A[tmem, BF16 pairs] * B[smem], K = 16 per instruction
__device__ __forceinline__ void mma_bf16_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(bdesc), "r"(idesc), "r"(acc)
        : "memory");
}
// MN-major operand with the 128-byte swizzle: rows of 64 elements along N,
// 8-row groups along K 1024 bytes apart (SBO), further 64 columns `lbo` on.
__device__ __forceinline__ uint64_t sdesc_sw128_mn(uint32_t saddr, uint32_t lbo) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((saddr >> 4) & 0x3fffu);
    d |= static_cast<uint64_t>(lbo >> 4) << 16;
    d |= static_cast<uint64_t>(1024u >> 4) << 32;
    d |= static_cast<uint64_t>(1u) << 46;
    d |= static_cast<uint64_t>(2u) << 61;
    return d;
}

// A role's place in the parts, task by task: a tile of a part of up to 128
// rows is one task, of a larger one two (its two MMA tiles on the same keys).
struct Task {
    int idx = -1, z = 0, t = 0, t0 = 0, t1 = 0, p0 = 0, n = 0, sub = 0;
    bool valid = false, pair = false;
    __device__ __forceinline__ bool fresh() const { return sub == 0; }             // the first task on its keys
    __device__ __forceinline__ bool done() const { return !pair || sub == 1; }     // the last
    __device__ __forceinline__ bool ends() const { return t == t1 - 1 && done(); }  // the part's last
    __device__ __forceinline__ bool tail() const { return (t + 1) * kKeys > p0; }  // holds keys behind the prefix
    __device__ __forceinline__ void next() {
        if (pair && sub == 0) {
            sub = 1;
        } else {
            sub = 0;
            ++t;
        }
    }
};
// What the converting (or cleaning) warps need of a tile.
struct TileInfo {
    int32_t what;       // kTileK, kTileV, kTileVTail, or kTileEnd: no more; BF16: the stage, or -1
    int32_t node, end;  // first key behind the prefix, and behind the sequence's rows, in keys of the tile
    int32_t idx;        // its part
};
enum : int { kTileK = 0, kTileV = 1, kTileVTail = 2, kTileEnd = 3 };

template <int D, bool FP8>
struct Geo {
    static constexpr int kStages = FP8 ? 3 : 4;         // BF16 K or V tiles
    static constexpr int kRaw = FP8 ? 3 : 0;            // E4M3 K or V tiles as loaded
    static constexpr int kTileBytes = kKeys * D * 2;    // also a Q tile's
    static constexpr int kRawBytes = kKeys * D;
    static constexpr int kHalf = kKeys * 128;           // 64 columns of a tile
    static constexpr int kQ = 0;
    static constexpr int kRing = 2 * kTileBytes;
    static constexpr int kRawAt = kRing + kStages * kTileBytes;
    static constexpr int kScaleAt = kRawAt + kRaw * kRawBytes;         // [stream][2][K | V][128] floats
    static constexpr int kMlAt = kScaleAt + (FP8 ? 2 * 2 * 2 * kKeys * 4 : 0);  // [stream][128] (m, l)
    static constexpr int kPartAt = kMlAt + 2 * kTileRows * 8;
    static constexpr int kInfoAt = kPartAt + kParts * static_cast<int>(sizeof(Part));
    static constexpr int kBarAt = kInfoAt + 4 * static_cast<int>(sizeof(TileInfo));
    static constexpr int kBars = 2 + 2 + 2 * kStages + 2 + 2 * (kRaw ? kRaw : 1) + 2 + 2 + 2 + 4 + 4 + 2 * kParts + 3;
    static constexpr int kSmem = 1024 + kBarAt + kBars * 8 + 64 + kBadRing * 4;
};

template <int D, bool FP8>
__global__ void __launch_bounds__(kThreads, 1) tree_attention_kernel(const __grid_constant__ CUtensorMap tmk,
                                                                     const __grid_constant__ CUtensorMap tmv,
                                                                     const __grid_constant__ TreeArgs a) {
    using G_ = Geo<D, FP8>;
    constexpr int NS = G_::kStages, NR = G_::kRaw ? G_::kRaw : 1;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bar = reinterpret_cast<uint64_t*>(sm + G_::kBarAt);
    uint64_t* q_full = bar;                 // row warp -> MMA, per Q slot
    uint64_t* q_empty = q_full + 2;
    uint64_t* kv_full = q_empty + 2;        // TMA (or the converting warps) -> MMA, per stage
    uint64_t* kv_empty = kv_full + NS;
    uint64_t* v_ask = kv_empty + NS;        // BF16: MMA -> cleaning warps, a tail tile of V is there
    uint64_t* v_fixed = v_ask + 1;          // and it is clean
    uint64_t* raw_full = v_fixed + 1;       // E4M3: TMA -> converting warps
    uint64_t* raw_empty = raw_full + NR;
    uint64_t* s_full = raw_empty + NR;      // per stream: scores ready
    uint64_t* p_full = s_full + 2;          // probabilities ready
    uint64_t* o_full = p_full + 2;          // a part's products complete
    uint64_t* sc_full = o_full + 2;         // scales of a task, [stream][2]
    uint64_t* sc_empty = sc_full + 4;
    uint64_t* pt_full = sc_empty + 4;       // part descriptors
    uint64_t* pt_empty = pt_full + kParts;
    uint64_t* ml_in = pt_empty + kParts;    // the streams' (m, l) exchanged
    uint64_t* ml_out = ml_in + 1;           // and both outputs read
    uint64_t* drained = ml_out + 1;         // after a time-out: no product in flight
    int* s_abort = reinterpret_cast<int*>(drained + 1);
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(s_abort + 1);
    int* s_bad = s_abort + 2; // [kBadRing] per part: a node's value is not finite
    __shared__ ShareScratch s_share;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < 2; ++s) {
            mbar_init(&q_full[s], 1);
            mbar_init(&q_empty[s], 1);
            mbar_init(&s_full[s], 1);
            mbar_init(&p_full[s], 4);
            mbar_init(&o_full[s], 1);
        }
        for (int s = 0; s < NS; ++s) {
            mbar_init(&kv_full[s], FP8 ? 4 : 1);
            mbar_init(&kv_empty[s], 1);
        }
        mbar_init(v_ask, 1);
        mbar_init(v_fixed, 4);
        for (int s = 0; s < NR; ++s) {
            mbar_init(&raw_full[s], 1);
            mbar_init(&raw_empty[s], 4);
        }
        for (int s = 0; s < 4; ++s) {
            mbar_init(&sc_full[s], 1);
            mbar_init(&sc_empty[s], 4);
        }
        for (int s = 0; s < kParts; ++s) {
            mbar_init(&pt_full[s], 1);
            mbar_init(&pt_empty[s], FP8 ? 11 : 10);  // TMA, MMA, 8 softmax warps, and the scale warp
        }
        mbar_init(ml_in, 8);
        mbar_init(ml_out, 8);
        mbar_init(drained, 1);
        *s_abort = 0;
        for (int s = 0; s < kBadRing; ++s) s_bad[s] = 0;
        fence_barrier_init();
        prefetch_tensormap(&tmk);
        prefetch_tensormap(&tmv);
        work_at(a.work).join[blockIdx.x].parts = 0;
        work_at(a.work).marks[blockIdx.x] = 0;
    }
    if (warp == kMmaWarp) tmem_alloc(s_tmem, 512);
    __syncthreads();
    pdl_trigger();  // the join's blocks may wait for this grid beside it

    Part* s_part = reinterpret_cast<Part*>(sm + G_::kPartAt);
    TileInfo* s_info = reinterpret_cast<TileInfo*>(sm + G_::kInfoAt);
    using ItemWalk = Walk<kItemRows, kKeys, 10, 2, 3>;
    // Weights in units of about 2,070 cycles, from the CTAs' times: a tile with two row tiles 6,200, with one 4,200, an
    // item's start and end 17,000 to 24,000.  With tiles alone a few CTAs took 1.5 times the others' (287 us above).
    // Taken from BF16 and E4M3 caches of D 128 and used for D 64 too, whose tiles are half as long.
    const Share share = find_share<D, kThreads, 1, ItemWalk>(a, s_share);
    const bool idle = share.lo >= share.hi;
    const uint32_t tmem = *s_tmem;
    volatile int* abort_flag = s_abort;
    tc_fence_after();

    // A bounded wait.  After a time-out no role waits, loads or multiplies any
    // more, and every role leaves at its next part.
    auto wait = [&](uint64_t* b, uint32_t parity) {
        if (mbar_try_wait(b, parity)) return;
        const uint64_t start = globaltimer_ns();
        while (!mbar_try_wait_sleep(b, parity, 100000u)) {
            if (*abort_flag) return;
            if (globaltimer_ns() - start > kWaitNs) *abort_flag = 1;
        }
    };
    // A role's next part; it hands a part's descriptor back when it is through with it.
    auto open = [&](Task& k) {
        ++k.idx;
        const int r = k.idx % kParts;
        wait(&pt_full[r], (k.idx / kParts) & 1u);
        const Part& p = s_part[r];
        k.valid = !*abort_flag && p.rows > 0;
        k.pair = p.rows > kTileRows;
        k.z = p.z;
        k.t = k.t0 = p.t0;
        k.t1 = p.t1;
        k.p0 = p.p0;
        k.n = p.n;
        k.sub = 0;
    };
    auto hand_back = [&](int idx) { mbar_arrive(&pt_empty[idx % kParts]); };
    // The order of a share's tiles, the same in every role: the scores are
    // taken two tasks ahead of the products with V, so K's tiles of tasks 0
    // and 1 come first, then V's of task u - 2 and K's of task u in turn.
    auto in_order = [&](auto&& on_v, auto&& on_k) {
        Task k, v1, v2;
        k.valid = true;
#pragma unroll 1
        for (uint32_t u = 0;; ++u) {
            if (k.valid && k.t == k.t1) open(k);
            if (v2.valid) on_v(v2, u - 2);
            if (k.valid) on_k(k, u);
            else if (!v1.valid) break;
            v2 = v1;
            v1 = k;
            if (k.valid) k.next();
        }
    };

    // the softmax warps take over the others' registers: 256 x 184 + 256 x 72 = 512 x 128
    if (warp >= kConvWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (idle) {
        // no share
    } else if (warp == kTmaWarp) {
        // ------------------------------------------------------------- loads
        if (lane == 0) {
            constexpr int N = FP8 ? NR : NS;
            uint64_t* full = FP8 ? raw_full : kv_full;
            uint64_t* empty = FP8 ? raw_empty : kv_empty;
            int count = 0;
            auto load = [&](const CUtensorMap* map, const Task& k, int what) {
                const int s = count % N;
                if (count >= N) wait(&empty[s], ((count / N) & 1u) ^ 1u);
                if (*abort_flag) return;
                if (FP8) {
                    s_info[s] = TileInfo{what, k.p0 - k.t * kKeys, k.p0 + k.n - k.t * kKeys, k.idx};
                    if (what == kTileEnd) {
                        mbar_arrive(&full[s]);
                        return;
                    }
                    mbar_arrive_expect_tx(&full[s], G_::kRawBytes);
                    tma_load_3d(sm + G_::kRawAt + s * G_::kRawBytes, map, &full[s], 0, k.t * kKeys, k.z);
                } else {
                    mbar_arrive_expect_tx(&full[s], G_::kTileBytes);
                    for (int h = 0; h < D / 64; ++h)
                        tma_load_3d(sm + G_::kRing + s * G_::kTileBytes + h * G_::kHalf, map, &full[s], 64 * h, k.t * kKeys, k.z);
                }
                ++count;
            };
            in_order(
                [&](const Task& v, uint32_t) {
                    if (v.fresh()) load(&tmv, v, v.tail() ? kTileVTail : kTileV);
                    if (v.ends()) hand_back(v.idx);
                },
                [&](const Task& k, uint32_t) {
                    if (k.fresh()) load(&tmk, k, kTileK);
                });
            if (FP8) load(&tmk, Task(), kTileEnd);
            if (*abort_flag)  // the copies in flight land before the CTA leaves
                for (int j = max(0, count - N); j < count; ++j) {
                    const uint64_t t = globaltimer_ns();
                    while (!mbar_try_wait(&full[j % N], (j / N) & 1u) && globaltimer_ns() - t < NF_WAIT_BUDGET_NS) {
                    }
                }
        }
    } else if (warp == kMmaWarp) {
        // ---------------------------------------------------------- products
        // Task u of the share belongs to stream u & 1.  Its scores are taken
        // two tasks ahead, behind the product with V of the task before in the
        // same stream, whose probabilities lie in the scores' columns.
        const uint32_t id_s = idesc_bf16(kTileRows, kKeys), id_o = idesc_bf16(kTileRows, D) | (1u << 16);
        const bool leader = elect_one() != 0;
        int count = 0, k_stage = 0, v_stage = 0, q_at = 0;
        uint32_t fixed = 0;
        auto entry = [&]() {  // the next tile of the ring
            const int s = count % NS;
            wait(&kv_full[s], (count / NS) & 1u);
            ++count;
            return s;
        };
        in_order(
            [&](const Task& v, uint32_t u) {
                const uint32_t s = u & 1;
                const bool clean = !FP8 && v.fresh() && v.tail();
                if (v.fresh()) v_stage = entry();
                if (clean && lane == 0) {
                    s_info[0] = TileInfo{v_stage, v.p0 - v.t * kKeys, v.p0 + v.n - v.t * kKeys, v.idx};
                    mbar_arrive(v_ask);
                }
                wait(&p_full[s], (u >> 1) & 1u);
                if (clean) wait(v_fixed, fixed++ & 1u);
                tc_fence_after();
                const bool start = v.pair ? v.t == v.t0 : v.t - v.t0 < 2;
                const bool last = v.pair ? v.t == v.t1 - 1 : v.t >= v.t1 - 2;
                if (leader && !*abort_flag) {
                    const uint64_t vd = sdesc_sw128_mn(smem_u32(sm + G_::kRing + v_stage * G_::kTileBytes), G_::kHalf);
#pragma unroll
                    for (int j = 0; j < kKeys / 16; ++j)
                        mma_bf16_ts(tmem + 256 + s * D, tmem + s * kKeys + j * 8, vd + j * (2048 >> 4), id_o, !(start && j == 0));
                    if (FP8 && v.tail())
#pragma unroll
                        for (int j = 0; j < kKeys / 16; ++j)
                            mma_bf16_ts(tmem + 256 + s * D, tmem + s * kKeys + kKeys / 2 + j * 8, vd + j * (2048 >> 4), id_o, 1);
                    if (v.done()) tc_commit(&kv_empty[v_stage]);
                    if (last) tc_commit(&o_full[s]);
                }
                __syncwarp();
                if (v.ends() && lane == 0) hand_back(v.idx);
            },
            [&](const Task& k, uint32_t u) {
                const int slot = (q_at + k.sub) & 1;
                if (k.t == k.t0) wait(&q_full[slot], ((q_at + k.sub) >> 1) & 1u);
                if (k.fresh()) k_stage = entry();
                tc_fence_after();
                if (leader && !*abort_flag) {
                    const uint64_t qd = sdesc_sw128(smem_u32(sm + G_::kQ + slot * G_::kTileBytes));
                    const uint64_t kd = sdesc_sw128(smem_u32(sm + G_::kRing + k_stage * G_::kTileBytes));
#pragma unroll
                    for (int j = 0; j < D / 16; ++j) {
                        const uint32_t off = ((j >> 2) * G_::kHalf + (j & 3) * 32) >> 4;
                        mma_bf16(tmem + (u & 1) * kKeys, qd + off, kd + off, id_s, j != 0);
                    }
                    tc_commit(&s_full[u & 1]);
                    if (k.done()) tc_commit(&kv_empty[k_stage]);
                    if (k.t == k.t1 - 1) tc_commit(&q_empty[slot]);
                }
                __syncwarp();
                if (k.ends()) q_at += k.pair ? 2 : 1;
            });
        if (!FP8 && lane == 0) {
            s_info[0].what = -1;
            mbar_arrive(v_ask);
        }
        if (*abort_flag && leader) {
            tc_commit(drained);
            const uint64_t t = globaltimer_ns();
            while (!mbar_try_wait(drained, 0) && globaltimer_ns() - t < NF_WAIT_BUDGET_NS) {
            }
        }
    } else if (warp == kRowWarp) {
        // ----------------------- the walk, and q's rows into swizzled tiles
        ItemWalk w;
        w.start(a, share, s_share);
        auto publish = [&](int idx) {
            const int r = idx % kParts;
            if (idx >= kParts) wait(&pt_empty[r], ((idx / kParts) & 1u) ^ 1u);
            if (lane == 0) {
                s_part[r] = w.describe(a, share);
                mbar_arrive(&pt_full[r]);
            }
            __syncwarp();
        };
        publish(0);
        int at = 0;
        for (int idx = 1; w.valid && !*abort_flag; ++idx) {
            // the next part is published first: its keys are on their way while these rows are fetched
            const int row0 = w.row0, all = w.rows;
            const uint16_t* q = a.q + (static_cast<int64_t>(w.first) * a.nq + w.g * a.G) * D;
            w.seek(a, false);
            publish(idx);
            constexpr int C = D / 8, S = 32 / C;  // 16-byte chunks of a row; rows at a time
            const int ch = lane % C;
            for (int r0 = 0; r0 < all; r0 += kTileRows, ++at) {
                const int slot = at & 1;
                if (at >= 2) wait(&q_empty[slot], ((at >> 1) & 1u) ^ 1u);
                const uint32_t dst = smem_u32(sm + G_::kQ + slot * G_::kTileBytes) + (ch >> 3) * G_::kHalf;
                int node = (row0 + r0 + lane / C) / a.G, h = row0 + r0 + lane / C - node * a.G;
                const int rows = min(kTileRows, all - r0);
#pragma unroll 4
                for (int r = lane / C; r < rows; r += S) {
                    const uint16_t* src = q + (static_cast<int64_t>(node) * a.nq + h) * D + ch * 8;
                    const uint32_t to = dst + r * 128 + (((ch & 7) ^ (r & 7)) << 4);
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(src) : "memory");
                    h += S;
                    while (h >= a.G) {
                        h -= a.G;
                        ++node;
                    }
                }
                asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_full[slot]);
            }
        }
    } else if (warp == kScaleWarp) {
        // ------------------- E4M3: a task's 128 key scales (times c) and value scales
        if (FP8) {
            Task k, prev;
            float ks[4], vs[4];
            k.valid = true;
#pragma unroll 1
            for (uint32_t u = 0;; ++u) {  // task u's scales are fetched, then those of task u - 1 stored
                float oks[4], ovs[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    oks[e] = ks[e];
                    ovs[e] = vs[e];
                }
                if (k.valid && k.t == k.t1) open(k);
                if (k.valid) {
                    const int64_t row = static_cast<int64_t>(k.z) * a.L;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = k.t * kKeys + 32 * e + lane;
                        const bool in = key < k.p0 + k.n;
                        ks[e] = in ? __ldg(a.k_scale + row + key) : 0.f;
                        vs[e] = in ? __ldg(a.v_scale + row + key) : 0.f;
                    }
                }
                if (u > 0) {
                    const uint32_t o = u - 1, at = 2 * (o & 1) + ((o >> 1) & 1);
                    if (o >= 4) wait(&sc_empty[at], ((o >> 2) & 1u) ^ 1u);
                    float* dst = reinterpret_cast<float*>(sm + G_::kScaleAt) + at * 2 * kKeys;
                    bool bad = false;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        dst[32 * e + lane] = oks[e] * a.c;
                        if (prev.t * kKeys + 32 * e + lane >= prev.p0 && !isfinite(ovs[e])) {
                            bad = true;
                            ovs[e] = 0.f;
                        }
                        dst[kKeys + 32 * e + lane] = ovs[e];
                    }
                    if (bad) s_bad[prev.idx % kBadRing] = 1;
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(&sc_full[at]);
                        if (prev.ends()) hand_back(prev.idx);
                    }
                }
                if (!k.valid) break;
                prev = k;
                k.next();
            }
        }
    } else {
        // E4M3: every tile to BF16.  BF16: the tail tiles of V, whose keys
        // behind the sequence's rows, and whose nodes' values that are not
        // finite, become zero (a zero probability must not meet a NaN).
        const int tid = threadIdx.x - kConvWarp * 32;
#pragma unroll 1
        for (int count = 0;; ++count) {
            if (FP8) {
                const int r = count % NR, s = count % NS;
                wait(&raw_full[r], (count / NR) & 1u);
                const TileInfo info = s_info[r];
                if (*abort_flag || info.what == kTileEnd) break;
                const bool tail = info.what == kTileVTail;
                const int node = info.node, end = info.end;
                uint8_t* dst = sm + G_::kRing + s * G_::kTileBytes;
                if (count >= NS) wait(&kv_empty[s], ((count / NS) & 1u) ^ 1u);
                const uint8_t* src = sm + G_::kRawAt + r * G_::kRawBytes;
                constexpr int C = D / 16;  // 16-byte chunks of a raw row
                bool bad = false;
                // chunk e of the raw tile (16 codes) to chunks 2 ch and 2 ch + 1 of its row; the upper half's threads
                // store the second first, so that eight threads' stores lie in eight bank groups
                auto put = [&](int e, const uint32_t* y) {
                    const int row = e / C, ch = e % C, flip = (ch >> 2) & 1;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int col = 2 * ch + (j ^ flip);
                        const bool up = (j ^ flip) != 0;
                        *reinterpret_cast<uint4*>(dst + (col >> 3) * G_::kHalf + row * 128 + (((col & 7) ^ (row & 7)) << 4)) =
                            up ? make_uint4(y[4], y[5], y[6], y[7]) : make_uint4(y[0], y[1], y[2], y[3]);
                    }
                };
                // exact, a NaN as a NaN: E4M3 -> F16 -> F32 -> BF16
                auto widen = [&](const uint4& x, uint32_t* y) {
                    const uint32_t in[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float lo, hi;
                            f16x2_to_f32(e4m3x2_to_f16x2(h ? in[j] >> 16 : in[j]), lo, hi);
                            y[2 * j + h] = bf16x2_hw(lo, hi);
                        }
                };
#pragma unroll 1
                for (int b = 0; b < C; b += 2) {
                    uint4 x[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) x[j] = *reinterpret_cast<const uint4*>(src + ((b + j) * 128 + tid) * 16);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        uint32_t y[8];
                        widen(x[j], y);
                        put((b + j) * 128 + tid, y);
                    }
                }
                if (__builtin_expect(tail, 0)) {
                    // V's rows behind the sequence, and a node's chunks that hold a NaN, become zeros
#pragma unroll 1
                    for (int e = tid; e < C * 128; e += 128) {
                        const int row = e / C;
                        const uint4 x = *reinterpret_cast<const uint4*>(src + e * 16);
                        uint32_t y[8] = {};
                        const uint32_t in[4] = {x.x, x.y, x.z, x.w};
                        uint32_t nan = 0;  // a code 0x7f carries into the sign's place
#pragma unroll
                        for (int j = 0; j < 4; ++j) nan |= ((in[j] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
                        const bool nan_node = nan != 0 && row >= node && row < end;
                        bad |= nan_node;
                        if (row >= end || nan_node) put(e, y);
                    }
                }
                if (bad) s_bad[info.idx % kBadRing] = 1;
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&raw_empty[r]);
                    mbar_arrive(&kv_full[s]);
                }
            } else {
                wait(v_ask, count & 1u);
                const TileInfo info = s_info[0];
                if (*abort_flag || info.what < 0) break;
                const int row = tid, node = info.node, end = info.end;
                uint8_t* dst = sm + G_::kRing + info.what * G_::kTileBytes;
                bool zero = row >= end;
                if (row >= node && row < end) {
                    uint32_t inf = 0;
#pragma unroll
                    for (int ch = 0; ch < D / 8; ++ch) {
                        const uint4 x = *reinterpret_cast<const uint4*>(dst + (ch >> 3) * G_::kHalf + row * 128 +
                                                                        (((ch & 7) ^ (row & 7)) << 4));
                        const uint32_t in[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j)  // an exponent of all ones carries into the sign's place
                            inf |= ((in[j] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
                    }
                    if (inf) {
                        zero = true;
                        s_bad[info.idx % kBadRing] = 1;
                    }
                }
                if (zero)
#pragma unroll
                    for (int ch = 0; ch < D / 8; ++ch)
                        *reinterpret_cast<uint4*>(dst + (ch >> 3) * G_::kHalf + row * 128 + (((ch & 7) ^ (row & 7)) << 4)) =
                            make_uint4(0u, 0u, 0u, 0u);
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(v_fixed);
            }
        }
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
        // ------------------------------------------- softmax of stream s
        const int s = warp >> 2, r = threadIdx.x & 127;  // the thread's row of the MMA tile
        const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;
        const uint32_t t_s = tmem + s * kKeys + lanes, t_o = tmem + 256 + s * D + lanes;
        float2* s_ml = reinterpret_cast<float2*>(sm + G_::kMlAt);
        uint32_t u0 = 0, mine_n = 0, o_n = 0, ml_n = 0;  // tasks before the part; this stream's tasks and parts; exchanges
        for (int idx = 0; !idle; ++idx) {
            wait(&pt_full[idx % kParts], (idx / kParts) & 1u);
            const Part& w = s_part[idx % kParts];
            if (*abort_flag || w.rows == 0) break;
            const int p0 = w.p0, n = w.n, t1 = w.t1;
            const bool pair = w.rows > kTileRows;
            const int mine0 = static_cast<int>((s ^ u0) & 1);  // pair: which MMA tile; else: the first tile's offset
            const int row0 = pair ? mine0 * kTileRows : 0;      // first row of the stream in the item
            const int rows = min(kTileRows, w.rows - row0);
            const bool active = (warp & 3) * 32 < rows;
            const int row = w.row0 + row0 + r, node = row / a.G;
            // A thread holds a quarter of the columns of rows lane / 4 and + 8 of either half (16 lanes) of the warp's
            // rows, as matrix fragments: so it needs 32 of a tile's 128 scales.  The half at hand's (max, sum) and the
            // other's change places.
            float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, mo[2] = {-INFINITY, -INFINITY}, lo[2] = {0.f, 0.f};
            const int mine_rows = rows - (warp & 3) * 32;  // rows of this warp
            int done = 0;
            for (int t = w.t0 + (pair ? 0 : mine0); t < t1; t += pair ? 1 : 2, ++mine_n, ++done) {
                const uint32_t b = mine_n & 1;
                const float* sc = reinterpret_cast<const float*>(sm + G_::kScaleAt) + (2 * s + b) * 2 * kKeys + 2 * (lane & 3);
                wait(&s_full[s], mine_n & 1u);
                if (FP8) wait(&sc_full[2 * s + b], (mine_n >> 1) & 1u);
                __syncwarp();
                tc_fence_after();
                // a tile with drafted keys has code of its own, so that the other's stays short
                auto half_rows = [&](int half, auto tail) {
                    constexpr bool kTail = decltype(tail)::value;
                    if (mine_rows > 16 * half) {
                        const uint32_t lane0 = static_cast<uint32_t>(half) << 20;
                        uint32_t v[64];
                        uint64_t nm[2];
                        auto pick = [&](int i, int h) {
                            return f32x2_pack(__uint_as_float(v[4 * i + 2 * h]), __uint_as_float(v[4 * i + 2 * h + 1]));
                        };
                        auto put = [&](int i, int h, uint64_t y) {
                            v[4 * i + 2 * h] = __float_as_uint(f32x2_lo(y));
                            v[4 * i + 2 * h + 1] = __float_as_uint(f32x2_hi(y));
                        };
                        auto factor = [&](int i) { return FP8 ? *reinterpret_cast<const uint64_t*>(sc + 8 * i) : f32x2_pack(a.c, a.c); };
                        auto negate = [&]() {
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const float mu = m[h] == -INFINITY ? 0.f : m[h];
                                nm[h] = f32x2_pack(-mu, -mu);
                            }
                        };
                        // v = x - m with the maxima brought up to date, and the sums and outputs with them
                        auto rise = [&]() {
                            tmem_ld_frag(t_s + lane0, v);
                            tmem_wait_ld();
                            // x = S * factor
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const uint64_t f = factor(i);
#pragma unroll
                                for (int h = 0; h < 2; ++h) put(i, h, mul_f32x2(pick(i, h), f));
                            }
                            if constexpr (kTail) {
                                const int ra = (warp & 3) * 32 + 16 * half + (lane >> 2);  // the thread's first row
#pragma unroll
                                for (int h = 0; h < 2; ++h) {
                                    const int nd = (w.row0 + row0 + ra + 8 * h) / a.G;
#pragma unroll
                                    for (int c = 0; c < 4; ++c) {
                                        const uint32_t vis = visible(a, w.first + nd, nd, n, t * kKeys + 32 * c - p0, ra + 8 * h < rows) >>
                                                             (2 * (lane & 3));
#pragma unroll
                                        for (int i = 0; i < 4; ++i)
#pragma unroll
                                            for (int e = 0; e < 2; ++e)
                                                if (!((vis >> (8 * i + e)) & 1u)) v[16 * c + 4 * i + 2 * h + e] = 0xff800000u;
                                    }
                                }
                            }
                            float mn[2], f[2];
                            bool grow = done == 0;
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                float mx[2] = {__uint_as_float(v[2 * h]), __uint_as_float(v[4 + 2 * h])};
#pragma unroll
                                for (int i = 0; i < 16; ++i)
                                    mx[i & 1] = max3(mx[i & 1], __uint_as_float(v[4 * i + 2 * h]), __uint_as_float(v[4 * i + 2 * h + 1]));
                                float x = fmaxf(mx[0], mx[1]);
                                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
                                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
                                mn[h] = fmaxf(m[h], x);
                                grow |= x > m[h] + kRescale;
                            }
                            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                                for (int h = 0; h < 2; ++h) {
                                    f[h] = m[h] == -INFINITY ? 0.f : ex2(m[h] - mn[h]);
                                    m[h] = mn[h];
                                    l[h] *= f[h];
                                }
                                // the products up to the previous task are complete: the scores' commit covers them
                                if (done > 0)
#pragma unroll 1
                                    for (int c = 0; c < D; c += 16) {
                                        uint32_t o[8];
                                        tmem_ld_frag16(t_o + lane0 + c, o);
                                        tmem_wait_ld();
#pragma unroll
                                        for (int k = 0; k < 8; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f[(k >> 1) & 1]);
                                        tmem_st_frag16(t_o + lane0 + c, o);
                                    }
                            }
                            negate();
#pragma unroll
                            for (int i = 0; i < 16; ++i)
#pragma unroll
                                for (int h = 0; h < 2; ++h) put(i, h, add_f32x2(pick(i, h), nm[h]));
                        };
                        if constexpr (kTail) {
                            rise();
                        } else {
                            // the maxima of the tiles before, as long as no weight gets beyond 2^kRescale with them
                            negate();
                            tmem_ld_frag(t_s + lane0, v);
                            tmem_wait_ld();
                            float top[2] = {m[0] == -INFINITY || m[1] == -INFINITY ? INFINITY : -INFINITY, -INFINITY};
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const uint64_t f = factor(i);
#pragma unroll
                                for (int h = 0; h < 2; ++h) {
                                    const uint64_t y = fma_f32x2(pick(i, h), f, nm[h]);
                                    put(i, h, y);
                                    top[h] = max3(top[h], f32x2_lo(y), f32x2_hi(y));
                                }
                            }
                            if (__builtin_expect(__any_sync(0xffffffffu, fmaxf(top[0], top[1]) > kRescale), 0)) rise();
                        }
                        uint32_t pk[32];
                        uint64_t sum[2] = {0, 0};
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            uint64_t g = 0;
                            if (FP8) g = *reinterpret_cast<const uint64_t*>(sc + kKeys + 8 * i);
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const uint64_t y = pick(i, h);
                                uint64_t pr = f32x2_pack(ex2(f32x2_lo(y)), ex2(f32x2_hi(y)));
                                sum[h] = add_f32x2(sum[h], pr);
                                if (FP8) pr = mul_f32x2(pr, g);
                                pk[2 * i + h] = bf16x2_hw(f32x2_lo(pr), f32x2_hi(pr));
                            }
                        }
                        tmem_st_pairs(t_s + lane0, pk);
                        if constexpr (FP8 && kTail) {
                            // What the rounding to BF16 leaves, for a second product: rows that see a few drafted keys
                            // would else carry the rounding of one key's scale in all their dims.
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const uint64_t g = *reinterpret_cast<const uint64_t*>(sc + kKeys + 8 * i);
#pragma unroll
                                for (int h = 0; h < 2; ++h) {
                                    const uint64_t y = pick(i, h);
                                    const uint64_t pr = mul_f32x2(f32x2_pack(ex2(f32x2_lo(y)), ex2(f32x2_hi(y))), g);
                                    const uint32_t hi = pk[2 * i + h];
                                    const float a0 = __uint_as_float(hi << 16), a1 = __uint_as_float(hi & 0xffff0000u);
                                    pk[2 * i + h] = bf16x2_hw(isinf(a0) ? 0.f : f32x2_lo(pr) - a0, isinf(a1) ? 0.f : f32x2_hi(pr) - a1);
                                }
                            }
                            tmem_st_pairs(t_s + lane0 + kKeys / 2, pk);
                        }
#pragma unroll
                        for (int h = 0; h < 2; ++h) l[h] += f32x2_lo(sum[h]) + f32x2_hi(sum[h]);  // of the thread's columns
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float tm = m[h], tl = l[h];
                        m[h] = mo[h];
                        l[h] = lo[h];
                        mo[h] = tm;
                        lo[h] = tl;
                    }
                };
                if ((t + 1) * kKeys > p0) {
#pragma unroll 1
                    for (int half = 0; half < 2; ++half) half_rows(half, std::true_type());
                } else {
#pragma unroll 1
                    for (int half = 0; half < 2; ++half) half_rows(half, std::false_type());
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&p_full[s]);
                    if (FP8) mbar_arrive(&sc_empty[2 * s + b]);
                }
            }
            // ------------------------------------------------ the part's end
            if (done > 0) {
                wait(&o_full[s], o_n & 1u);
                ++o_n;
                __syncwarp();
                tc_fence_after();
            }
            // from the fragments' rows to the thread's own, r
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                float x = h < 2 ? l[h & 1] : lo[h & 1];
                x += __shfl_xor_sync(0xffffffffu, x, 1);
                x += __shfl_xor_sync(0xffffffffu, x, 2);
                if ((lane & 3) == 0)
                    s_ml[s * kTileRows + (warp & 3) * 32 + 8 * h + (lane >> 2)] = make_float2(h < 2 ? m[h & 1] : mo[h & 1], x);
            }
            __syncwarp();
            const float mr = s_ml[s * kTileRows + r].x;
            float lr = s_ml[s * kTileRows + r].y;
            if (__any_sync(0xffffffffu, s_bad[idx % kBadRing] != 0))
                if (poisoned<D, FP8>(a, w.z, p0, n, w.first, node, r < rows)) {
                    lr = NAN;
                    s_ml[s * kTileRows + r].y = lr;
                }
            __syncwarp();
            const bool whole = w.kind == 3;
            const int slot = 2 * blockIdx.x + (w.kind & 1), cnt = t1 - w.t0;
            const Work wk = work_at(a.work);
            float other_m = -INFINITY, other_l = 0.f;
            if (!pair) {
                // both streams hold parts of the same rows: exchange (m, l), then each finishes half of the columns
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(ml_in);
                wait(ml_in, ml_n & 1u);
                __syncwarp();
                tc_fence_after();
                const float2 o = s_ml[(s ^ 1) * kTileRows + r];
                other_m = o.x;
                other_l = o.y;
            }
            if (active) {
                const float mt = fmaxf(mr, other_m), mu = mt == -INFINITY ? 0.f : mt;
                const float f0 = mr == -INFINITY ? 0.f : ex2(mr - mu), f1 = other_m == -INFINITY ? 0.f : ex2(other_m - mu);
                const float lt = lr * f0 + other_l * f1;
                const bool use0 = done > 0, use1 = !pair && cnt - done > 0;
                const float inv = lt == 0.f ? 0.f : 1.f / lt;
                const uint32_t t_other = tmem + 256 + (s ^ 1) * D + lanes;
                const int irow = row0 + r;  // the thread's row in the item
                uint16_t* dst = a.out + (static_cast<int64_t>(w.first + node) * a.nq + w.g * a.G + (row - node * a.G)) * D;
                float* part_o = wk.acc + (static_cast<int64_t>(slot) * kItemRows + irow) * D;
                for (int c = (pair ? 0 : s * D / 64); c < (pair ? D / 32 : (s + 1) * D / 64); ++c) {
                    uint32_t v[32];
                    float o[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j) o[j] = 0.f;
                    if (use0) {
                        tmem_ld32(t_o + 32 * c, v);
                        tmem_wait_ld();
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] = __uint_as_float(v[j]) * f0;
                    }
                    if (use1) {
                        tmem_ld32(t_other + 32 * c, v);
                        tmem_wait_ld();
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] = fmaf(__uint_as_float(v[j]), f1, o[j]);
                    }
                    if (r < rows) {
                        if (whole) {
#pragma unroll
                            for (int j = 0; j < 16; ++j) v[j] = bf16x2_hw(o[2 * j] * inv, o[2 * j + 1] * inv);
#pragma unroll
                            for (int j = 0; j < 16; j += 4)
                                *reinterpret_cast<uint4*>(dst + 32 * c + 2 * j) = make_uint4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                        } else {
#pragma unroll
                            for (int j = 0; j < 32; j += 8)
                                st_global_v8(part_o + 32 * c + j, __float_as_uint(o[j]), __float_as_uint(o[j + 1]),
                                             __float_as_uint(o[j + 2]), __float_as_uint(o[j + 3]), __float_as_uint(o[j + 4]),
                                             __float_as_uint(o[j + 5]), __float_as_uint(o[j + 6]), __float_as_uint(o[j + 7]));
                        }
                    }
                }
                if (!whole && r < rows && (pair || s == 0)) wk.ml[static_cast<int64_t>(slot) * kItemRows + irow] = make_float2(mu, lt);
            }
            __syncwarp();
            tc_fence_before();
            if (!pair) {  // no product into the streams' outputs before both have read them
                if (lane == 0) mbar_arrive(ml_out);
                wait(ml_out, ml_n++ & 1u);
            }
            if (r == 0) s_bad[(idx + kBadRing / 2) % kBadRing] = 0;
            u0 += pair ? 2 * cnt : cnt;
            __syncwarp();
            if (lane == 0) hand_back(idx);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
    if (threadIdx.x == 0 && *abort_flag) {
        work_at(a.work).marks[blockIdx.x] = kMarkGaveUp;
        if (a.status) atomicCAS(a.status, 0, NF_DEVERR_WAIT_FULL);
    }
}

// NaN into `rows` rows of the output from `first` on, shared by all threads of the grid.
template <int D>
__device__ __forceinline__ void fill_nan(const TreeArgs& a, int first, int rows) {
    const int64_t per_row = static_cast<int64_t>(a.nq) * D, n = rows * per_row / 8;
    uint4* dst = reinterpret_cast<uint4*>(a.out + first * per_row);
    const int64_t threads = static_cast<int64_t>(gridDim.x) * gridDim.y * blockDim.x;
    int64_t e = (static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * blockDim.x + threadIdx.x;
#pragma unroll 1
    for (; e < n; e += threads) dst[e] = make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
}
// What the join does beside joining, with all threads of its grid: the rows of refused sequences become NaN (4,096 rows of
// 32 heads of 128: 24 us; one thread of the attention's took 384 ms), and after a wait that ran out, when nothing of
// the call can be relied on, every row does.  Returns whether that is so.
template <int D>
__device__ __forceinline__ bool rows_without_result(const TreeArgs& a, const Work& wk) {
    static_assert(kMaxCtas <= 256);
    const int mark = threadIdx.x < gridDim.x ? wk.marks[threadIdx.x] : 0;
    if (__builtin_expect(!__syncthreads_or(mark), 1)) return false;
    if (__syncthreads_or(mark == kMarkGaveUp)) {
        const int first = min(max(a.row_start[0], 0), a.rows), end = min(max(a.row_start[a.batch], 0), a.rows);
        fill_nan<D>(a, first, max(0, end - first));
        return true;
    }
    // a block looks at 256 sequences at a time, a thread each, and then takes its share of every bad one's rows
    __shared__ int2 s_rows[256];
    __shared__ int s_n;
#pragma unroll 1
    for (int i0 = 0; i0 < a.batch; i0 += 256) {
        __syncthreads();
        if (threadIdx.x == 0) s_n = 0;
        __syncthreads();
        Walk<kItemRows, kKeys, 0, 1, 1> w;  // (for its view of a sequence)
        w.i = i0 + static_cast<int>(threadIdx.x);
        if (w.i < a.batch) {
            w.load(a);
            if (w.n > 0 && w.bad(a)) s_rows[atomicAdd(&s_n, 1)] = make_int2(w.first, w.n);
        }
        __syncthreads();
#pragma unroll 1
        for (int k = 0; k < s_n; ++k) fill_nan<D>(a, s_rows[k].x, s_rows[k].y);
    }
    return false;
}

// Joins the parts of items that several CTAs computed, in their order: two
// rows a warp and two parts at a time, which is 1.3 us less than four and four (24 sequences x 16 nodes, 8191 keys).
constexpr int kJoinRows = 16;  // rows of a block
template <int D>
__global__ void __launch_bounds__(256) tree_join_kernel(const __grid_constant__ TreeArgs a) {
    pdl_wait();
    const Work wk = work_at(a.work);
    const int b = blockIdx.x;
    const JoinDesc d = wk.join[b];
    if (rows_without_result<D>(a, wk)) return;
    const int lane = threadIdx.x & 31, r0 = blockIdx.y * kJoinRows + (threadIdx.x >> 5) * 2;
    if (d.parts == 0 || r0 >= d.rows) return;
    constexpr int E = D / 32;
    // part 0 lies in slot 2 b + 1, part i > 0 in slot 2 (b + i)
    auto slot = [&](int i, int r) { return static_cast<int64_t>(i == 0 ? 2 * b + 1 : 2 * (b + i)) * kItemRows + r0 + r; };
    float m[2], l[2], acc[2][E];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[r][e] = 0.f;
        if (r0 + r < d.rows)
            for (int i = lane; i < d.parts; i += 32) {
                const float2 v = wk.ml[slot(i, r)];
                if (v.y != 0.f) m[r] = fmaxf(m[r], v.x);  // a part in which the row sees a key
            }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m[r] = fmaxf(m[r], __shfl_xor_sync(0xffffffffu, m[r], o));
#pragma unroll 1
    for (int i0 = 0; i0 < d.parts; i0 += 2) {
        float2 v[2][2];
        float p[2][2][E];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const bool in = i0 + i < d.parts && r0 + r < d.rows;
                v[i][r] = in ? wk.ml[slot(i0 + i, r)] : make_float2(0.f, 0.f);
                const float* src = wk.acc + slot(i0 + i, r) * D + lane * E;
                if (E == 4) {
                    const float4 x = in ? *reinterpret_cast<const float4*>(src) : make_float4(0.f, 0.f, 0.f, 0.f);
                    p[i][r][0] = x.x;
                    p[i][r][1] = x.y;
                    p[i][r][E - 2] = x.z;
                    p[i][r][E - 1] = x.w;
                } else {
                    const float2 x = in ? *reinterpret_cast<const float2*>(src) : make_float2(0.f, 0.f);
                    p[i][r][0] = x.x;
                    p[i][r][1] = x.y;
                }
            }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float f = v[i][r].y != 0.f ? ex2(v[i][r].x - m[r]) : 0.f;
                l[r] += v[i][r].y * f;
#pragma unroll
                for (int e = 0; e < E; ++e) acc[r][e] += f == 0.f ? 0.f : p[i][r][e] * f;
            }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        if (r0 + r >= d.rows) continue;
        const int row = d.row0 + r0 + r, node = row / a.G;
        uint16_t* dst = a.out + (static_cast<int64_t>(d.first + node) * a.nq + d.head * a.G + (row - node * a.G)) * D + lane * E;
        const float inv = l[r] == 0.f ? 0.f : 1.f / l[r];
        if (E == 4)
            *reinterpret_cast<uint2*>(dst) = make_uint2(bf16x2_hw(acc[r][0] * inv, acc[r][1] * inv),
                                                        bf16x2_hw(acc[r][E - 2] * inv, acc[r][E - 1] * inv));
        else
            *reinterpret_cast<uint32_t*>(dst) = bf16x2_hw(acc[r][0] * inv, acc[r][1] * inv);
    }
}

// The same for items of few rows, a warp a row, in little code: such a call's
// time is its latency, and much of that the first run through each instruction.
template <int D>
__global__ void __launch_bounds__(256) tree_join_few_kernel(const __grid_constant__ TreeArgs a) {
    pdl_wait();
    const Work wk = work_at(a.work);
    const int b = blockIdx.x;
    const JoinDesc d = wk.join[b];
    if (rows_without_result<D>(a, wk)) return;
    const int lane = threadIdx.x & 31, r = blockIdx.y * 8 + (threadIdx.x >> 5);
    if (d.parts == 0 || r >= d.rows) return;
    constexpr int E = D / 32;
    float m = -INFINITY, l = 0.f, acc[E] = {};
#pragma unroll 4
    for (int i = 0; i < d.parts; ++i) {
        const int64_t at = static_cast<int64_t>(i == 0 ? 2 * b + 1 : 2 * (b + i)) * kItemRows + r;
        const float2 v = wk.ml[at];
        float x[E];
        if (E == 4) *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(wk.acc + at * D + lane * E);
        else *reinterpret_cast<float2*>(x) = *reinterpret_cast<const float2*>(wk.acc + at * D + lane * E);
        if (v.y == 0.f) continue;  // the row sees no key of this part
        const float mn = fmaxf(m, v.x), f0 = ex2(m - mn), f1 = ex2(v.x - mn);
        m = mn;
        l = l * f0 + v.y * f1;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = acc[e] * f0 + x[e] * f1;
    }
    const int row = d.row0 + r, node = row / a.G;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint32_t* dst = reinterpret_cast<uint32_t*>(
        a.out + (static_cast<int64_t>(d.first + node) * a.nq + d.head * a.G + (row - node * a.G)) * D + lane * E);
#pragma unroll
    for (int e = 0; e < E; e += 2) dst[e / 2] = bf16x2_hw(acc[e] * inv, acc[e + 1] * inv);
}

template <int D, bool FP8>
cudaError_t launch_many(const nf_kv_cache& c, const TreeArgs& a, int grid, cudaStream_t st) {
    CUtensorMap tmk, tmv;
    const uint64_t heads = static_cast<uint64_t>(c.seqs) * c.kv_heads;
    if (!make_tmap_kv(&tmk, c.k, !FP8, D, c.max_context, heads, kKeys) ||
        !make_tmap_kv(&tmv, c.v, !FP8, D, c.max_context, heads, kKeys))
        return cudaErrorInvalidValue;
    static bool attr[kMaxDevices] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
    constexpr int smem = Geo<D, FP8>::kSmem;
    if (!attr[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(tree_attention_kernel<D, FP8>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        attr[dev] = true;
    }
    tree_attention_kernel<D, FP8><<<grid, kThreads, smem, st>>>(tmk, tmv, a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_tree_attention(const nf_kv_cache& c, const uint16_t* q, int rows, int q_heads,
                                  const int32_t* row_start, int batch, const int32_t* prefix, const int32_t* cache_seq,
                                  const uint64_t* mask, int mask_words, float scale, uint16_t* out, void* work,
                                  int32_t* status, cudaStream_t st) {
    if (rows <= 0 || batch <= 0) return cudaSuccess;
    TreeArgs a{};
    a.q = q;
    a.out = out;
    a.row_start = row_start;
    a.prefix = prefix;
    a.cache_seq = cache_seq;
    a.mask = mask;
    a.k_scale = c.k_scale;
    a.v_scale = c.v_scale;
    a.v = c.v;
    a.work = work;
    a.status = status;
    a.rows = rows;
    a.nq = q_heads;
    a.nkv = c.kv_heads;
    a.G = q_heads / c.kv_heads;
    a.batch = batch;
    a.seqs = c.seqs;
    a.L = c.max_context;
    a.words = mask_words;
    a.c = scale * 1.4426950408889634f;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
    static int sms[kMaxDevices] = {};
    if (!sms[dev]) sms[dev] = std::min(kMaxCtas, gemm_grid_size(dev));
    const int grid = sms[dev];
    const bool fp8 = c.kind == NF_KV_E4M3, wide = c.head_dim == 128;
    // By the rows that a sequence has per KV head, on average; any choice is right for any rows.  Measured (us, 32
    // sequences on 4,000 keys, D 128, 4 KV heads, keys from DRAM) with items of 8 rows, 16 rows, and the kernel for many:
    //   rows      8             16            24            32            64
    //   E4M3  37.9 52.2 66.6  48.1 56.3 66.6  54.3 62.5 72.7  72.7 74.8 72.7  130 114 72.7
    //   BF16  50.2 52.2 60.4  58.4 54.3 62.4  74.8 62.5 62.5  97.3 72.7 62.5  175 114 64.5
    // and one sequence on 65,000 keys: E4M3, 32 rows: 62.5 64.5 72.7; BF16, 24 rows: 80.9 68.6 70.7.  E4M3's keys take
    // longer to convert than a second look at them in the L2.
    // The average serves a batch of one length.  255 sequences of one row on 1,000 to 2,000 keys and a chunk behind 32,768
    // less its rows, in one call and apart: a chunk of 512 rows (all in items of 8 or 16 rows) E4M3 2,510 against 85 + 423,
    // BF16 2,040 against 133 + 315; of 1,024 (E4M3 and BF16 in the kernel for many) 1,110 against 85 + 822, 785 against
    // 133 + 587.  A caller with such a batch does better with two calls.
    const int64_t all = static_cast<int64_t>(rows) * a.G;
    const int nt = all <= (fp8 ? 32ll : 8ll) * batch ? 1 : !fp8 && all <= 24ll * batch ? 2 : 0;
    cudaError_t e = nt    ? launch_tree_few(c, a, nt, grid, st)
                    : fp8 ? (wide ? launch_many<128, true>(c, a, grid, st) : launch_many<64, true>(c, a, grid, st))
                          : (wide ? launch_many<128, false>(c, a, grid, st) : launch_many<64, false>(c, a, grid, st));
    if (e == cudaSuccess)
        e = nt ? launch_dependent(wide ? tree_join_few_kernel<128> : tree_join_few_kernel<64>, dim3(grid, nt), dim3(256), 0, st, a)
               : launch_dependent(wide ? tree_join_kernel<128> : tree_join_kernel<64>, dim3(grid, kItemRows / kJoinRows),
                                  dim3(256), 0, st, a);
    return e;
}

}  // namespace nf

using namespace nf;

extern "C" {

int64_t nf_tree_attention_workspace(int head_dim) {
    if (head_dim != 64 && head_dim != 128) return 0;
    return kJoinBytes + kMarkBytes + kMlBytes + 2ll * kMaxCtas * kItemRows * head_dim * 4;
}

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
