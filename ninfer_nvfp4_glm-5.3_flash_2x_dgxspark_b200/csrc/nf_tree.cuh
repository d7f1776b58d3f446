// nf_tree.cuh -- what the two kernels of nf_tree_attention share: the division
// of the work, the masks, and the parts that are joined.
//
// The rows of a sequence and KV head are its nodes' q heads of that group, R =
// nodes * G rows (row = node * G + head): one pass over the keys serves them
// all.  With c = scale * log2 e, row r and key j:
//   x = c q_r . k_j (times the key's scale),  m = running max of x,
//   p = 2^(x - m),  l = sum p,  O = sum p v_j (times the value's scale)
// and the result is O / l.  Parts of the keys give (m, l, O) each, and
// O = sum O_i 2^(m_i - m), l = sum l_i 2^(m_i - m) joins them.
#pragma once

#include "nf_kv.h"

#include "nf_common.cuh"
#include "nf_gemm_shared.cuh"
#include "nf_internal.h"

namespace nf {

constexpr int kStatusBad = NF_DEVERR_BAD_TOKEN;
constexpr int kTileRows = 128;   // rows per tcgen05 tile
constexpr int kItemRows = 256;   // most rows of a work item
constexpr int kMaxCtas = 148;    // CTAs (one per SM) the workspace has parts for
constexpr int kParts = 8;        // part descriptors in flight
constexpr uint64_t kWaitNs = 10000000000ull;  // some waits last as long as a whole part

// What the join's kernel needs of an item in several parts: written by the CTA
// of its first part.
struct JoinDesc {
    int32_t parts;   // 0: nothing to join
    int32_t rows;    // rows of the item
    int32_t row0;    // its first row (node * G + head) in the sequence
    int32_t first;   // the sequence's first row of q
    int32_t head;    // KV head
    int32_t pad[3];
};
enum : int32_t { kMarkGaveUp = 1, kMarkRefused = 2 };  // a wait of the CTA ran out; some sequence is refused
struct Work {
    JoinDesc* join;  // [kMaxCtas]
    int32_t* marks;  // [kMaxCtas]: what the join has to know of every CTA
    float2* ml;      // [2 kMaxCtas][kItemRows] (m, l)
    float* acc;      // [2 kMaxCtas][kItemRows][D]
};
constexpr int64_t kJoinBytes = (kMaxCtas * sizeof(JoinDesc) + 255) / 256 * 256;
constexpr int64_t kMarkBytes = (kMaxCtas * 4 + 255) / 256 * 256;
constexpr int64_t kMlBytes = 2ll * kMaxCtas * kItemRows * 8;

__host__ __device__ inline Work work_at(void* p) {
    uint8_t* b = static_cast<uint8_t*>(p);
    uint8_t* parts = b + kJoinBytes + kMarkBytes;
    return Work{reinterpret_cast<JoinDesc*>(b), reinterpret_cast<int32_t*>(b + kJoinBytes), reinterpret_cast<float2*>(parts),
                reinterpret_cast<float*>(parts + kMlBytes)};
}

struct TreeArgs {
    const uint16_t* q;
    uint16_t* out;
    const int32_t* row_start;
    const int32_t* prefix;
    const int32_t* cache_seq;
    const uint64_t* mask;
    const float* k_scale;
    const float* v_scale;
    const void* v;  // the values once more, for the rare look at single rows
    void* work;
    int32_t* status;
    int rows, nq, nkv, G, batch, seqs, L, words;
    float c;        // scale * log2(e)
};

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t codes) {  // the low two codes
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(codes)));
    return r;
}
// Which of 32 keys the row of a node sees: the keys are the sequence's rows
// j .. j + 31 (below 0: the prefix), of n rows; qrow is the node's row of q.
__device__ __forceinline__ uint32_t visible(const TreeArgs& a, int64_t qrow, int node, int n, int j, bool valid) {
    auto low = [](int k) { return k >= 32 ? ~0u : k <= 0 ? 0u : (1u << k) - 1u; };
    if (!a.mask) return low(min(n, node + 1) - j);
    uint64_t bits = 0;
    if (j > -32 && valid) {
        const unsigned long long* mw = reinterpret_cast<const unsigned long long*>(a.mask) + qrow * a.words;
        const int wi = j >> 6, sh = j & 63;
        if (wi >= 0 && wi < a.words) bits = __ldg(mw + wi) >> sh;
        if (sh > 32 && wi + 1 >= 0 && wi + 1 < a.words) bits |= __ldg(mw + wi + 1) << (64 - sh);
    }
    return (static_cast<uint32_t>(bits) & low(n - j)) | low(-j);
}
// Which of the sequence's rows j .. j + 31 hold a value that is not finite, a row a lane of the whole warp.
template <int D, bool FP8>
__device__ __forceinline__ uint32_t bad_values(const TreeArgs& a, int z, int p0, int n, int j) {
    j += static_cast<int>(threadIdx.x & 31);
    bool bad = false;
    if (j < n) {
        const int64_t at = static_cast<int64_t>(z) * a.L + p0 + j;
        if (FP8) bad = !isfinite(a.v_scale[at]);
        const uint4* v = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.v) + at * D * (FP8 ? 1 : 2));
#pragma unroll 4
        for (int c = 0; c < D * (FP8 ? 1 : 2) / 16; ++c) {
            const uint4 x = v[c];
            const uint32_t in[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int k = 0; k < 4; ++k)  // an exponent of all ones (E4M3: 0x7f) carries into the sign's place
                bad |= FP8 ? (((in[k] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0
                           : (((in[k] & 0x7f807f80u) + 0x00800080u) & 0x80008000u) != 0;
        }
    }
    return __ballot_sync(0xffffffffu, bad);
}
// Whether a lane's node sees a row of the sequence whose value is not finite; looked at only when some row's is, by whole
// warps, so that each row's values are read once a warp (a chunk of 200 BF16 rows among 150 single ones, a NaN in its last
// row's value: 146 us instead of 87; each thread for itself 65,000).
template <int D, bool FP8>
__device__ __noinline__ bool poisoned(const TreeArgs& a, int z, int p0, int n, int first, int node, bool valid) {
    bool seen = false;
#pragma unroll 1
    for (int j = 0; j < n; j += 32) {
        const uint32_t bad = bad_values<D, FP8>(a, z, p0, n, j);
        if (bad != 0) seen |= (visible(a, static_cast<int64_t>(first) + node, node, n, j, valid) & bad) != 0;
    }
    return valid && seen;
}

// A part as the kernels' roles see it; rows 0 ends the share.
struct Part {
    int32_t z;      // cache sequence * KV heads + KV head
    int32_t t0, t1; // its tiles
    int32_t p0, n;  // the sequence's prefix and rows
    int32_t first;  // the sequence's first row of q
    int32_t row0, rows;  // the item's rows (node * G + head) of the sequence
    int32_t g;      // KV head
    int32_t kind;   // bit 0: holds tile 0, bit 1: holds the last tile
    int32_t pad[2];
};

// A CTA's share [lo, hi) of the line, whose CTAs take `per` each.
struct Share {
    int64_t per, lo, hi;
};
struct ShareScratch {
    int64_t base, head;  // weight before the share's first sequence, and of one of that one's heads
    int64_t warp[32];
    int32_t seq;
};

// ---------------------------------------------------------------------------
// The work: every (sequence, KV head, up to ROWS rows) is an item of ceil(keys
// / KEYS) tiles.  An item weighs ITEM, for its start and end, and a tile ONE, or
// TWO when the item's rows fill two tcgen05 tiles.  The items in order
// (sequence, head, rows) form one line of weight, each item's ITEM before its
// tiles, which the CTAs cut into equal shares; a tile belongs to the share in
// which it starts.  So the SMs get the same work whatever the lengths, and a long
// sequence is cut into as many parts as it has shares.  One warp walks through
// the parts of the CTA's share and publishes them to the others in a ring of
// descriptors.
// ---------------------------------------------------------------------------
template <int ROWS, int KEYS, int ITEM, int ONE, int TWO>
struct Walk {
    static constexpr int kTile = ONE > TWO ? ONE : TWO;  // the most that a tile weighs
    // the sequence
    int i, first, n, p0, sq, npt;
    // the part: rows [row0, row0 + rows) of KV head g, tiles [t0, t1) of kt
    int g, pt, t0, t1, kt, row0, rows, keys;
    int64_t at, lo, hi;  // weight at the item's start, and the CTA's share
    bool valid;

    __device__ __forceinline__ bool pair() const { return rows > kTileRows; }

    __device__ __forceinline__ void load(const TreeArgs& a) {
        first = min(max(__ldg(a.row_start + i), 0), a.rows);
        n = max(0, min(max(__ldg(a.row_start + i + 1), 0), a.rows) - first);
        p0 = __ldg(a.prefix + i);
        sq = a.cache_seq ? __ldg(a.cache_seq + i) : i;
        npt = (n * a.G + ROWS - 1) / ROWS;
    }
    __device__ __forceinline__ bool bad(const TreeArgs& a) const {
        return p0 < 0 || sq < 0 || sq >= a.seqs || p0 > a.L - n;
    }
    // shape of item pt of the sequence
    __device__ __forceinline__ void item(const TreeArgs& a) {
        row0 = pt * ROWS;
        rows = min(ROWS, n * a.G - row0);
        keys = p0 + (a.mask ? n : min(n, (row0 + rows - 1) / a.G + 1));
        kt = (keys + KEYS - 1) / KEYS;
    }
    // where the item's tile t starts, from the item's start, and the first tile that starts at `w` or behind it
    __device__ __forceinline__ int64_t tile_at(int t) const { return ITEM + static_cast<int64_t>(t) * (pair() ? TWO : ONE); }
    __device__ __forceinline__ int tile_from(int64_t w) const {
        const int64_t x = max(w - ITEM, static_cast<int64_t>(0));
        return static_cast<int>(min(static_cast<int64_t>(kt), pair() ? (x + TWO - 1) / TWO : (x + ONE - 1) / ONE));
    }
    __device__ __forceinline__ int64_t weight() const { return tile_at(kt); }
    // weight of the sequence's items of one head
    __device__ __forceinline__ int64_t head_weight(const TreeArgs& a) {
        int64_t w = 0;
#pragma unroll 1
        for (pt = 0; pt < npt; ++pt) {
            item(a);
            w += weight();
        }
        return w;
    }
    // the share's first part
    __device__ __forceinline__ void start(const TreeArgs& a, const Share& s, const ShareScratch& sh) {
        valid = true;
        i = sh.seq;
        lo = s.lo;
        hi = s.hi;
        load(a);
        g = static_cast<int>((lo - sh.base) / sh.head);
        at = sh.base + g * sh.head;
        pt = 0;
        seek(a, true);
    }
    // the part's descriptor, and, for an item that other CTAs go on with, what its join needs
    __device__ __forceinline__ Part describe(const TreeArgs& a, const Share& s) const {
        Part p{};
        if (!valid) return p;
        p.z = sq * a.nkv + g;
        p.t0 = t0;
        p.t1 = t1;
        p.p0 = p0;
        p.n = n;
        p.first = first;
        p.row0 = row0;
        p.rows = rows;
        p.g = g;
        p.kind = (t0 == 0) | (t1 == kt) << 1;
        if (p.kind == 1) {
            JoinDesc d{};
            d.parts = static_cast<int>((at + tile_at(kt - 1)) / s.per) - static_cast<int>(blockIdx.x) + 1;
            d.rows = rows;
            d.row0 = row0;
            d.first = first;
            d.head = g;
            work_at(a.work).join[blockIdx.x] = d;
        }
        return p;
    }
    // from the item (g, pt) at weight `at` to the first part inside the share, that item's own among them if `here`
    __device__ __forceinline__ void seek(const TreeArgs& a, bool here) {
#pragma unroll 1
        for (;; here = false) {
            if (!here) {
                at += weight();
                if (at >= hi) {
                    valid = false;
                    return;
                }
                if (++pt == npt) {
                    pt = 0;
                    if (++g == a.nkv) {
                        g = 0;
#pragma unroll 1
                        do {
                            ++i;  // at < hi <= total: there is another sequence with items
                            load(a);
                        } while (n == 0 || bad(a));
                    }
                }
            }
            item(a);
            t0 = tile_from(lo - at);
            t1 = tile_from(hi - at);
            if (t0 < t1) return;
        }
    }
};

// Finds the CTA's share (every thread sums the weights of a run of sequences) and marks bad sequences for the join.  A share
// is not smaller than LEAST tiles, those that a CTA takes at a time: smaller
// ones would only make more parts to join, and no share inside an item may be
// without a tile.  Ends with a __syncthreads.
template <int D, int THREADS, int LEAST, typename W>
__device__ __forceinline__ Share find_share(const TreeArgs& a, ShareScratch& sh) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    W w;
    const int run = (a.batch + THREADS - 1) / THREADS;
    const int i0 = min(a.batch, static_cast<int>(threadIdx.x) * run), i1 = min(a.batch, i0 + run);
    int64_t mine = 0;
#pragma unroll 1
    for (w.i = i0; w.i < i1; ++w.i) {
        w.load(a);
        if (w.n == 0) continue;
        if (w.bad(a)) {
            if (a.status) atomicCAS(a.status, 0, kStatusBad);
            work_at(a.work).marks[blockIdx.x] = kMarkRefused;
            continue;
        }
        mine += w.head_weight(a) * a.nkv;
    }
    int64_t before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += up;
    }
    if (lane == 31) sh.warp[warp] = before;
    __syncthreads();
    int64_t total = 0, base = before - mine;
#pragma unroll 1
    for (int k = 0; k < THREADS / 32; ++k) {
        if (k < warp) base += sh.warp[k];
        total += sh.warp[k];
    }
    Share s;
    s.per = max((total + gridDim.x - 1) / gridDim.x, static_cast<int64_t>(LEAST * W::kTile));
    s.lo = s.per * blockIdx.x;
    s.hi = min(total, s.lo + s.per);
    if (mine > 0 && s.lo >= base && s.lo < base + mine) {
#pragma unroll 1
        for (w.i = i0; w.i < i1; ++w.i) {
            w.load(a);
            if (w.n == 0 || w.bad(a)) continue;
            const int64_t here = w.head_weight(a);
            sh.head = here;
            if (s.lo < base + here * a.nkv) break;
            base += here * a.nkv;
        }
        sh.seq = w.i;
        sh.base = base;
    }
    __syncthreads();
    return s;
}

// The kernel for few rows (nf_tree_few.cu), with items of up to 8 nt rows; E4M3: nt 1.
cudaError_t launch_tree_few(const nf_kv_cache& c, const TreeArgs& a, int nt, int grid, cudaStream_t st);

}  // namespace nf
