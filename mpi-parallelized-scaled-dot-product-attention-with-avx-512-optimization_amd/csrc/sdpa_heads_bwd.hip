// sdpa_heads_bwd.hip -- gradients of attention_window, and the weights every key was given (attention_scored).
//
//     P = exp(s - lse) on visible pairs, dP = dO V^T, delta_i = sum_d dO_id O_id = sum_j P_ij dP_ij, dS = P * (dP - delta)
//     dV = P^T dO      dK = scale dS^T Q (both summed over the G heads that share them)      dQ = scale dS K
//
// Two kernels, no atomics: one whose workgroups own query rows (dQ, and delta on the way), one whose workgroups own keys (dK, dV)
// and walk the rows that see them -- the rows of a key head are its tokens' grouped heads, so the sum over a group is part of
// the walk.  P is computed in both (two products more than the five a single pass needs) because the alternative, adding dQ
// contributions of key blocks in memory, would make the result depend on the order of atomics.
#include "sdpa_heads_device.h"

namespace sdpa {
namespace heads {
namespace {

__device__ inline const char *row_at(const sdpa_tensor &t, long b, long tok, long head, int elem) {
    return (const char *)t.data + (b * t.batch + tok * t.token + head * t.head) * elem;
}

// 4 consecutive gradients of a row
template <typename T>
__device__ inline void store_grad(const sdpa_tensor &t, int b, int tok, int head, int d, int dim, bool vec, f32x4 v) {
    T *row = (T *)t.data + b * t.batch + tok * t.token + head * t.head;
    if (vec) {
        if (d >= dim) return;
        union { T e[4]; uint64_t u; f32x4 f; } y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y.e[i] = from_f32<T>(v[i]);
        if (sizeof(T) == 2) *reinterpret_cast<uint64_t *>(row + d) = y.u;
        else *reinterpret_cast<f32x4 *>(row + d) = y.f;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (d + i < dim) row[d + i] = from_f32<T>(v[i]);
    }
}

template <typename T, int DP>
__device__ inline void load_row(typename Ops<T>::Frag *f, const void *row, int dim, bool live, bool vec, int lane) {
#pragma unroll
    for (int s = 0; s < DP / Ops<T>::kStep; ++s) {
        union { u32x4 u; typename Ops<T>::Frag f; } y;
        y.u = u32x4{0, 0, 0, 0};
        if (live) y.u = load_chunk((const T *)row, s * Ops<T>::kStep + (lane >> 5) * Ops<T>::kVec, dim, vec);
        f[s] = y.f;
    }
}

// ---- one 32 x 32 block of pairs -------------------------------------------------------------------------------------------------
// Tiles X and Y lie in LDS (X = Q, Y = dO against a wave's keys; X = K, Y = V against a wave's queries), their partners x and y in
// registers, one column to a lane:
//     S = X x,  dP = Y y,  P = exp(S - lse),  dS = P * (dP - delta),   then   acc_y += Y^T P  (dV)   and   acc_x += X^T dS  (dK or dQ).
// Written down unit by unit (see Pipe): the exponentials stand beside the units of dP, the rest beside those of dV; dP begins at -delta.
// What a lane's column sees of the block's rows r: r < hi and (r >= lo or r < sk).
struct Sees { int hi, lo, sk; };

// lse and -delta: of the lane's column (rows kernel) or of the block's rows, in LDS (keys kernel)
struct ColumnStats {
    float lse2, neg_delta;
    __device__ f32x4 lse_at(int) const { return f32x4{lse2, lse2, lse2, lse2}; }
    __device__ f32x4 delta_at(int) const { return f32x4{neg_delta, neg_delta, neg_delta, neg_delta}; }
};
struct RowStats {
    unsigned at;                                        // + the lane half's 16 bytes; -delta lies 256 bytes behind lse
    __device__ f32x4 lse_at(int i) const { return lds_read<f32x4>(at, i * 32); }
    __device__ f32x4 delta_at(int i) const { return lds_read<f32x4>(at, 256 + i * 32); }
};

template <typename T, int DP, bool VY, bool VX, bool MASKED, typename Stats> struct GradBlock {
    using Frag = typename Ops<T>::Frag;
    static constexpr int KU = DP / Ops<T>::kStep, VK = sizeof(T) == 2 ? 2 : 4, VU = DP / 32 * VK;
    static constexpr int B0 = KU, C0 = B0 + (VX ? KU : 0), D0 = C0 + (VY ? VU : 0), UNITS = D0 + (VX ? VU : 0), AHEAD = 3;
    unsigned xr, yr, xc, yc;                            // where the lane reads the tiles' rows and columns
    Frag ring[AHEAD + 1];
    f32x16 s, dp;
    f32x4 lse[4];
    Probs<T> p, ds;
    uint32_t vis;
    __device__ inline __attribute__((always_inline)) Frag fetch(int u) const {
        if (u < B0) return read_rows<T, DP>(xr, 0, u);
        if (u < C0) return read_rows<T, DP>(yr, 0, u - B0);
        if (u < D0) return read_cols_part<DP>(yc, 0, (u - C0) / VK, (u - C0) % VK, T());
        return read_cols_part<DP>(xc, 0, (u - D0) / VK, (u - D0) % VK, T());
    }
    __device__ inline __attribute__((always_inline)) void weight(int i, float scale) {
        s[i] = __builtin_amdgcn_exp2f(s[i] * scale - lse[i >> 2][i & 3]);
        if (MASKED) s[i] = (vis >> i) & 1 ? s[i] : 0.f;
        if (VY && (sizeof(T) == 4 || (i & 1))) put_prob(p, s, i);
    }
    __device__ inline __attribute__((always_inline)) void slope(int i) {
        s[i] = MASKED && !((vis >> i) & 1) ? 0.f : s[i] * dp[i];
        if (sizeof(T) == 4 || (i & 1)) put_prob(ds, s, i);
    }
    template <int U>
    __device__ inline __attribute__((always_inline)) void unit(f32x16 *ax, f32x16 *ay, const Frag *x, const Frag *y, float scale) {
        if constexpr (U < UNITS) {
            if constexpr (U + AHEAD < UNITS) ring[(U + AHEAD) % (AHEAD + 1)] = fetch(U + AHEAD);
            const Frag f = ring[U % (AHEAD + 1)];
            if constexpr (U == C0 && !VX) {             // (nothing to stand beside)
#pragma unroll
                for (int i = 0; i < 16; ++i) weight(i, scale);
            }
            if constexpr (U == D0 && VX && !VY) {
#pragma unroll
                for (int i = 0; i < 16; ++i) slope(i);
            }
            if constexpr (U < B0) s = Ops<T>::mma(f, x[U], s);
            else if constexpr (U < C0) dp = Ops<T>::mma(f, y[U - B0], dp);
            else if constexpr (U < D0) ay[(U - C0) / VK] = mma_part(f, p, (U - C0) % VK, ay[(U - C0) / VK]);
            else ax[(U - D0) / VK] = mma_part(f, ds, (U - D0) % VK, ax[(U - D0) / VK]);
            if constexpr (VX && U > B0 && U < C0) {      // (one unit behind the product they read)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (B0 + 1 + i * (KU - 1) / 16 == U) weight(i, scale);
            }
            if constexpr (VX && VY && U > C0 && U < D0) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (C0 + 1 + i * (VU - 1) / 16 == U) slope(i);
            }
            __builtin_amdgcn_sched_barrier(0);
            unit<U + 1>(ax, ay, x, y, scale);
        }
    }
    __device__ inline __attribute__((always_inline)) void begin(unsigned tx, unsigned ty, const LaneMap<T, DP> &map, const Stats &st, Sees see) {
        xr = tx + map.rows; yr = ty + map.rows; xc = tx + map.cols; yc = ty + map.cols;
        s = f32x16{};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            lse[i] = st.lse_at(i);
            if (VX) {
                const f32x4 d = st.delta_at(i);
#pragma unroll
                for (int k = 0; k < 4; ++k) dp[4 * i + k] = d[k];
            }
        }
        if (MASKED) {
            vis = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int r = row_of(i, 0);
                vis |= r < see.hi && (r >= see.lo || r < see.sk) ? 1u << i : 0u;
            }
        }
    }
    __device__ inline __attribute__((always_inline)) void run(f32x16 *ax, f32x16 *ay, const Frag *x, const Frag *y, unsigned tx, unsigned ty,
                                                              const LaneMap<T, DP> &map, const Stats &st, Sees see, float scale) {
        begin(tx, ty, map, st, see);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) ring[u] = fetch(u);
        __builtin_amdgcn_sched_barrier(0);
        unit<0>(ax, ay, x, y, scale);
    }
    // the same arithmetic with products that leave out what a masked pair holds (block_not_finite)
    __device__ inline __attribute__((always_inline)) void run_guarded(f32x16 *ax, f32x16 *ay, const Frag *x, const Frag *y, unsigned tx, unsigned ty,
                                                                      const LaneMap<T, DP> &map, const Stats &st, Sees see, float scale, int lane) {
        begin(tx, ty, map, st, see);
#pragma unroll
        for (int i = 0; i < KU; ++i) s = Ops<T>::mma(read_rows<T, DP>(xr, 0, i), x[i], s);
#pragma unroll
        for (int i = 0; i < 16; ++i) weight(i, scale);
        if constexpr (VY) mma_block<T, DP, DP / 32>(ay, ty, map, 0, p, true, vis, 1, lane);
        if constexpr (VX) {
#pragma unroll
            for (int i = 0; i < KU; ++i) dp = Ops<T>::mma(read_rows<T, DP>(yr, 0, i), y[i], dp);
#pragma unroll
            for (int i = 0; i < 16; ++i) slope(i);
            mma_block<T, DP, DP / 32>(ax, tx, map, 0, ds, true, vis, 1, lane);
        }
    }
};

// The rows a key head's queries are walked in: blocks of 32, whole tokens' grouped heads to a block (the rows a block has left
// over are zeros), or, for groups of more than 32 heads, blocks of one token.  So a row's place inside its block is the same in
// every block, and a tile of blocks costs the DMA no vector arithmetic.
struct RowBlocks {
    int G, tokens, split;                               // tokens of a block, blocks of a token: one of them is 1
    __device__ explicit RowBlocks(int g) : G(g), tokens(g <= 32 ? 32 / g : 1), split(g <= 32 ? 1 : (g + 31) / 32) {}
    __device__ int row(int t) const { return (split > 1 ? t * split : t / tokens) * 32 + (split > 1 ? 0 : t % tokens * G); }
    __device__ int token(int block, int i) const { return split > 1 ? block / split : block * tokens + i / G; }
    __device__ int head(int block, int i) const { return split > 1 ? block % split * 32 + i : i % G; }
    __device__ bool used(int block, int i) const { return split > 1 ? head(block, i) < G : i < tokens * G; }
};

// delta of rows that see few keys, as the sum of P dP it stands for: sum dO * O takes O as it was rounded, which a mean over many keys
// hides and one over few does not.  bf16, 16 heads on 4 of 128 columns, dQ off by (of its norm) and the call's time, sum dO * O -> sum P dP:
// 15 keys a row 0.0021 -> 0.00166, 49 -> 50 us; 150 keys 0.00186 -> 0.00166, 78 -> 84; 1024 keys with the sum for the first rows only
// 0.00168, 395 us, and for all of them 0.00166, 477 us.  One walk more over tiles that lie in the L2.
constexpr int kDeltaKeys = 512;
template <typename T, int DP>
__device__ inline float weighted_sum(const typename Ops<T>::Frag *q, const typename Ops<T>::Frag *g, unsigned tk, unsigned tv,
                                     const LaneMap<T, DP> &map, float lse2, Sees see, float scale) {
    f32x16 s = {}, dp = {};
#pragma unroll
    for (int i = 0; i < DP / Ops<T>::kStep; ++i) s = Ops<T>::mma(read_rows<T, DP>(tk + map.rows, 0, i), q[i], s);
#pragma unroll
    for (int i = 0; i < DP / Ops<T>::kStep; ++i) dp = Ops<T>::mma(read_rows<T, DP>(tv + map.rows, 0, i), g[i], dp);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int r = row_of(i, 0);
        const bool seen = r < see.hi && (r >= see.lo || r < see.sk);
        sum += seen ? __builtin_amdgcn_exp2f(s[i] * scale - lse2) * dp[i] : 0.f;
    }
    return sum;
}

// ---- dQ: 128 rows to a workgroup, 32 to a wave -------------------------------------------------------------------------
// Two sequences of 4096 tokens, 16 heads on 4 of 128 columns, window 1024, bf16: 149 us, 91 GFLOP in three products = 610 TFLOP/s.  Counters:
// matrix instructions (dS is two operands) 0.39 of a SIMD's cycles, vector ones 0.28, a wave waits 0.29 of its time and has no turn for 0.32.
template <typename T, int DP, int BN, bool VEC>
__global__ __launch_bounds__(kHeadsThreads, DP * (int)sizeof(T) <= 256 ? 2 : 1)
void backward_rows_kernel(BackwardArgs a, int rows, int G, int tiles) {
    using TL = Tile<T, DP>;
    constexpr int STEPS = DP / Ops<T>::kStep, TILE = BN * TL::kRowBytes;
    __shared__ __attribute__((aligned(1024))) char lds[4 * TILE];            // K, V, K, V
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int id = xcd_place(blockIdx.x, gridDim.x);
    const int tile = tiles - 1 - id % tiles;
    id /= tiles;
    const int h = id % a.Hkv, b = id / a.Hkv;
    const int nq = clamp_len(a.q_lens, b, a.Tq), nk = clamp_len(a.kv_lens, b, a.Tk);
    const int r0 = tile * 128, rw = r0 + wave * 32, r = rw + (lane & 31);
    const int t = r / G, hq = h * G + r - t * G;
    const bool live = r < rows && t < nq;
    const SeenRange wg = seen_range(r0 / G, min(r0 + 127, rows - 1) / G, nq, nk, a.window);
    const SeenRange wv = seen_range(rw / G, min(rw + 31, rows - 1) / G, nq, nk, a.window);
    const Seen seen = live ? seen_at(nk - nq + t, nk, a.window) : Seen{0, 0};
    const KeyList list = key_list(wg, a.sinks);
    const int count = list.tiles(BN);
    Stager<T, DP, BN, 4> sk, sv;
    sk.init(row_at(a.k, b, 0, h, sizeof(T)), a.k.token, a.Dk, wave, lane);
    sv.init(row_at(a.v, b, 0, h, sizeof(T)), a.v.token, a.Dv, wave, lane);
    if (VEC && (a.Dk < DP || a.Dv < DP)) {
        zero_lds(lds, 4 * TILE, kHeadsThreads);
        __syncthreads();
    }
    const unsigned lds0 = lds_address(lds);
    auto stage = [&](int it, int buf) {
        if (VEC) {
            sk.dma(lds0 + buf * 2 * TILE, it * BN, list, wave, lane);
            sv.dma(lds0 + buf * 2 * TILE + TILE, it * BN, list, wave, lane);
        } else {
            sk.copy(lds + buf * 2 * TILE, it * BN, list, wave, lane);
            sv.copy(lds + buf * 2 * TILE + TILE, it * BN, list, wave, lane);
        }
    };
    if (count > 0) stage(0, 0);

    typename Ops<T>::Frag q[STEPS], g[STEPS];
    load_row<T, DP>(q, row_at(a.q, b, t, hq, sizeof(T)), a.Dk, live, a.vec, lane);
    load_row<T, DP>(g, row_at(a.dout, b, t, hq, sizeof(T)), a.Dv, live, a.vec, lane);
    const long at = ((long)b * a.Hq + hq) * a.Tq + t;
    const float lse2 = live ? a.lse[at] * kLog2e : __builtin_inff();     // (a row that does not exist: weight 2^(0 - inf) = 0)
    LaneMap<T, DP> map;
    map.init(lane);
    auto sees = [&](Frame f) {
        const int at = f.j0 + 4 * (opaque(lane) >> 5);
        return Sees{seen.hi - at, seen.lo - at, f.sinks - at};
    };
    float delta = 0.f;
    if (sizeof(T) == 2 && list.n <= kDeltaKeys) {        // (the first tile is on its way)
#pragma unroll 1
        for (int it = 0; it < count; ++it) {
            if (it > 0) {
                __syncthreads();
                stage(it, 0);
            }
            dma_wait();
            __syncthreads();
#pragma unroll 1
            for (int n = 0; n < BN / 32; ++n) {
                const Frame f = list.frame(it * BN + n * 32, 32);
                if (!sees_some(wv, f, 32)) continue;
                const unsigned tk = lds0 + n * 32 * TL::kRowBytes;
                delta += weighted_sum<T, DP>(q, g, tk, tk + TILE, map, lse2, sees(f), a.scale_log2);
            }
        }
        delta = half_sum(delta);
        __syncthreads();
        if (count > 1) stage(0, 0);
    } else {
        const T *row = (const T *)row_at(a.out, b, t, hq, sizeof(T));
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            union { u32x4 u; typename Ops<T>::Frag f; } y;
            y.u = u32x4{0, 0, 0, 0};
            if (live) y.u = load_chunk(row, s * Ops<T>::kStep + (lane >> 5) * Ops<T>::kVec, a.Dv, a.vec);
#pragma unroll
            for (int i = 0; i < Ops<T>::kVec; ++i) delta += to_f32(y.f[i]) * to_f32(g[s][i]);
        }
        delta = half_sum(delta);
    }
    if (r < rows && lane < 32) {                         // for the keys kernel, in the order it walks the rows
        const RowBlocks rb(G);
        const int g = r - t * G, place = rb.row(t) + g;
        float *l = a.stats + ((long)b * a.Hkv + h) * a.stat_rows + place;
        const int used = rb.split > 1 ? (g == G - 1 ? g & 31 : 31) : rb.tokens * G - 1;
        const int fill = (place & 31) == used ? 32 - (place & 31) : 1;     // (with the last row of a block, what the block has left over)
        for (int i = 0; i < fill; ++i) {
            l[i] = i == 0 ? lse2 : __builtin_inff();
            l[a.stat_stride + i] = i == 0 ? -delta : 0.f;
        }
    }

    f32x16 dq[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) dq[d][i] = 0.f;
    const ColumnStats stats = {lse2, -delta};
    bool odd = false;                                    // a block with masked pairs holds values that are no numbers
    // Blocks in order, those without a masked pair in a loop of their own: with both kinds in one loop the compiler keeps the accumulators in
    // different registers on the two paths and moves all of them in every turn.
    constexpr int PER = BN / 32;
    const int total = count * PER;
    auto arrive = [&](int e) {
        if (e % PER != 0) return;
        dma_wait();
        __syncthreads();
        if (e / PER + 1 < count) stage(e / PER + 1, (e / PER + 1) & 1);
    };
    auto tile_of = [&](int e) { return lds0 + (e / PER & 1) * 2 * TILE + e % PER * 32 * TL::kRowBytes; };
    auto whole = [&](int e) { return sees_all(wv, list.frame(e * 32, 32), 32); };
    int e = 0;
    while (e < total) {
#pragma unroll 1
        for (; e < total && !whole(e); ++e) {
            arrive(e);
            const Frame f = list.frame(e * 32, 32);
            if (!sees_some(wv, f, 32)) continue;
            const unsigned tk = tile_of(e), tv = tk + TILE;
            odd = odd || block_not_finite<T, DP>(tk, 0, lane);
            GradBlock<T, DP, false, true, true, ColumnStats> blk;
            blk.run(dq, nullptr, q, g, tk, tv, map, stats, sees(f), a.scale_log2);
        }
#pragma unroll 1
        for (; e < total && whole(e); ++e) {
            arrive(e);
            const unsigned tk = tile_of(e), tv = tk + TILE;
            GradBlock<T, DP, false, true, false, ColumnStats> blk;
            blk.run(dq, nullptr, q, g, tk, tv, map, stats, Sees{}, a.scale_log2);
        }
    }
    if (__syncthreads_or(odd)) {                          // then the workgroup does its rows once more, with guarded products
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) dq[d][i] = 0.f;
#pragma unroll 1
        for (int it = 0; it < count; ++it) {
            __syncthreads();
            stage(it, 0);
            dma_wait();
            __syncthreads();
#pragma unroll 1
            for (int n = 0; n < BN / 32; ++n) {
                const Frame f = list.frame(it * BN + n * 32, 32);
                if (!sees_some(wv, f, 32)) continue;
                const unsigned tk = lds0 + n * 32 * TL::kRowBytes, tv = tk + TILE;
                GradBlock<T, DP, false, true, true, ColumnStats> blk;
                blk.run_guarded(dq, nullptr, q, g, tk, tv, map, stats, sees(f), a.scale_log2, lane);
            }
        }
    }
    if (r >= rows) return;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f32x4 v;
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = live ? dq[d][4 * i + k] * a.scale : 0.f;
            store_grad<T>(a.dq, b, t, hq, d * 32 + 8 * i + 4 * (lane >> 5), a.Dk, a.vec_out, v);
        }
}

// slots of a key block's partial gradients (1: it writes the gradients itself), and of the blocks before it
__device__ inline int block_slots(const BackwardArgs &a, int block) { return a.chunks + (block < a.sink_blocks ? a.tail_chunks : 0); }
__device__ inline long slots_before(const BackwardArgs &a, int block) {
    const long n = a.chunks > 1 || block < a.sink_blocks ? block : a.sink_blocks;      // (blocks of one slot take no place)
    const int sinks = block < a.sink_blocks ? block : a.sink_blocks;
    return a.tail_chunks == 0 && a.chunks == 1 ? 0 : n * a.chunks + (long)sinks * a.tail_chunks;
}

// which queries see a key: tokens [lo, hi)
struct SeenBy { int lo, hi; };
__device__ inline SeenBy seen_by(int j, int nq, int nk, int window, int sinks) {
    SeenBy s = {0, 0};
    if (j >= nk || nq <= 0) return s;
    const int p0 = nk - nq;                             // the first query's position (below 0: it has seen nothing yet)
    const int lo = j - p0 > 0 ? j - p0 : 0;
    const int hi = j < sinks || j - p0 + window > nq ? nq : j - p0 + window;
    if (hi <= lo) return s;
    s.lo = lo; s.hi = hi;
    return s;
}

// Tiles of two such blocks of one tensor, staged by four waves
template <typename T, int DP> struct RowStager {
    using TL = Tile<T, DP>;
    static constexpr int kPieces = 64 * TL::kRowBytes / 1024 / 4;
    const char *base;
    long token, head;
    int dim;
    unsigned off[kPieces];
    __device__ static int row(int wave, int lane, int k) { return ((wave * kPieces + k) * 1024 + lane * 16) / TL::kRowBytes; }
    __device__ static int source(int wave, int lane, int k) {
        return (((wave * kPieces + k) * 64 + lane) % TL::kChunks) ^ TL::swz(row(wave, lane, k));
    }
    __device__ void init(const void *p, const sdpa_tensor &t, int d, const RowBlocks &rb, int wave, int lane) {
        base = uniform((const char *)p);
        token = t.token * (long)sizeof(T);
        head = t.head * (long)sizeof(T);
        dim = d;
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
            const int r = row(wave, lane, k), i = r & 31;
            off[k] = (unsigned)(((r >> 5) * rb.tokens + i / rb.G) * (int)token + i % rb.G * (int)head) + 16u * (unsigned)source(wave, lane, k);
        }
    }
    // (groups of at most 32 heads) rows behind the last query are read as the last query's: their weights are masked.  -> true: exactly
    // kPieces instructions are on their way
    __device__ bool dma(unsigned lds, int block, int nq, const RowBlocks &rb, int wave, int lane) const {
        const int t0 = block * rb.tokens;
        const char *at = base + (long)t0 * token;
        lds += (unsigned)(wave * kPieces) * 1024u;
        if (dim == DP && rb.tokens * rb.G == 32 && t0 + 2 * rb.tokens <= nq) {
#pragma unroll
            for (int k = 0; k < kPieces; ++k) lds_dma(at, off[k], lds + k * 1024u);
            return true;
        }
        const int ln = opaque(lane);
#pragma unroll 1
        for (int k = 0; k < kPieces; ++k) {
            const int r = row(wave, ln, k), i = r & 31, x = (r >> 5) * rb.tokens + i / rb.G, c = source(wave, ln, k);
            const unsigned o = (unsigned)((t0 + x < nq ? x : nq - 1 - t0) * (int)token + i % rb.G * (int)head) + 16u * (unsigned)c;
            if (i < rb.tokens * rb.G && c * Ops<T>::kVec < dim) lds_dma(at, o, lds + k * 1024u);      // (the rest stays zero)
        }
        return false;
    }
    __device__ void copy(char *tile, int block, int nq, const RowBlocks &rb, bool vec, int wave, int lane) const {
#pragma unroll 4
        for (int k = 0; k < kPieces; ++k) {
            const int ln = opaque(lane), r = row(wave, ln, k), blk = block + (r >> 5), i = r & 31, t = rb.token(blk, i);
            u32x4 x = {0, 0, 0, 0};
            if (t < nq && rb.used(blk, i))
                x = load_chunk(reinterpret_cast<const T *>(base + t * token + rb.head(blk, i) * head), source(wave, ln, k) * Ops<T>::kVec, dim, vec);
            *reinterpret_cast<u32x4 *>(tile + (wave * kPieces + k) * 1024 + ln * 16) = x;
        }
    }
};

// ---- dK, dV: 64 keys to a workgroup -----------------------------------------------------------------------------------------
// Waves 0 and 1 take 32 keys each on the even row blocks, waves 2 and 3 the same keys on the odd ones; the two sums are added in LDS
// at the end.  The shape above: 290 us, 121 GFLOP in four products = 420 TFLOP/s.  Counters: matrix instructions (P and dS are two operands)
// 0.30 of a SIMD's cycles, vector ones 0.20, LDS 0.14 of a CU's, 0.18 idle behind the last round of workgroups, and the one wave of
// a SIMD (accumulators and operands fill the registers) waits 0.32 of its time: every block starts with reads and a chain of products that
// nothing stands beside.  With P and dS in one term, 237 us then: 128 keys to a workgroup of eight waves, V in LDS in place of
// registers, took 286; -lse / scale and -delta as the products' start, for fewer vector instructions, 245.
// WHAT: 3 = both; heads of 256 do them one after the other (1 = dV, 2 = dK): two accumulators and two operands of 256 columns leave
// no registers for the scores.
template <typename T, int DP, int WHAT, bool VEC>
__global__ __launch_bounds__(kHeadsThreads, DP * (int)sizeof(T) <= 128 ? 2 : 1)
void backward_keys_kernel(BackwardArgs a, int G, int blocks) {
    using TL = Tile<T, DP>;
    constexpr int STEPS = DP / Ops<T>::kStep, TILE = 64 * TL::kRowBytes;
    constexpr int NBUF = 131072 / (2 * TILE) < 4 ? 131072 / (2 * TILE) : 4, AHEAD = NBUF - 1, PIECES = 2 * RowStager<T, DP>::kPieces;
    constexpr bool DV = (WHAT & 1) != 0, DK = (WHAT & 2) != 0;
    __shared__ __attribute__((aligned(1024))) char lds[2 * TILE * NBUF];     // Q, dO, Q, dO
    __shared__ __attribute__((aligned(16))) float lstat[NBUF][2][64];         // [buffer][lse, -delta][row]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // the blocks' walks over the rows that see them by the window first, then the short ones over the rows that see only their sinks
    const int groups = a.B * a.Hkv, plain = blocks * a.chunks;
    const bool tail = (int)blockIdx.x >= groups * plain;
    int id = tail ? (int)blockIdx.x - groups * plain : xcd_place(blockIdx.x, groups * plain);
    const int per = tail ? a.sink_blocks * a.tail_chunks : plain, chunks = tail ? a.tail_chunks : a.chunks;
    const int item = id % per, block = item / chunks, chunk = item % chunks;
    id /= per;
    const int h = id % a.Hkv, b = id / a.Hkv;
    const int nq = clamp_len(a.q_lens, b, a.Tq), nk = clamp_len(a.kv_lens, b, a.Tk);
    const int k0 = block * kBwdKeys, kw = k0 + (wave & 1) * 32, phase = wave >> 1, j = kw + (lane & 31);
    const RowBlocks rb(G);

    // the tokens that see any of the workgroup's keys: contiguous, from the first key's first to the last key's last (or, with a sink key
    // among them, to the end)
    const int klast = min(k0 + kBwdKeys, nk) - 1;
    SeenBy all = {0, 0};
    if (k0 < nk && nq > 0) {
        const SeenBy first = seen_by(k0, nq, nk, a.window, a.sinks), last = seen_by(klast, nq, nk, a.window, a.sinks);
        all.lo = max(0, k0 - (nk - nq));
        all.hi = max(first.hi, last.hi);
    }
    const SeenBy tok = seen_by(j, nq, nk, a.window, a.sinks);
    const SeenBy by = {rb.row(tok.lo), tok.hi > tok.lo ? rb.row(tok.hi) : 0};
    // rows that see every key of the wave: from the last key's first to the smallest end, which is the first key's that is no sink
    SeenBy full = {0, 0};
    if (kw + 32 <= nk) {
        const SeenBy f = seen_by(kw < a.sinks ? min(a.sinks, kw + 31) : kw, nq, nk, a.window, a.sinks);
        const SeenBy l = seen_by(kw + 31, nq, nk, a.window, a.sinks);
        if (f.hi > 0 && l.hi > 0) full = SeenBy{rb.row(l.lo), rb.row(min(f.hi, l.hi))};
    }
    const int blk0 = rb.row(all.lo) / 64 * 2;            // row blocks come in pairs
    const int pairs = all.hi > all.lo ? ((rb.row(all.hi) + 31) / 32 - blk0 + 1) / 2 : 0;
    int begin = 0, end = pairs;                           // a sink block: the pairs its window reaches, and behind them the tail
    if (block < a.sink_blocks && a.tail_chunks > 0) {
        const SeenBy w = seen_by(klast, nq, nk, a.window, 0);
        const int reach = w.hi > w.lo ? min(pairs, max(0, ((rb.row(w.hi) + 31) / 32 - blk0 + 1) / 2)) : 0;
        begin = tail ? reach : 0;
        end = tail ? pairs : reach;
    }
    const int it0 = begin + (int)((long)(end - begin) * chunk / chunks), it1 = begin + (int)((long)(end - begin) * (chunk + 1) / chunks);
    const bool idle = tail && kw >= a.sinks;              // (a tail's rows see nothing else)

    RowStager<T, DP> sq, sg;
    sq.init(row_at(a.q, b, 0, h * G, sizeof(T)), a.q, a.Dk, rb, wave, lane);
    sg.init(row_at(a.dout, b, 0, h * G, sizeof(T)), a.dout, a.Dv, rb, wave, lane);
    if (VEC && (a.Dk < DP || a.Dv < DP || rb.tokens * G < 32)) {
        zero_lds(lds, 2 * TILE * NBUF, kHeadsThreads);
        __syncthreads();
    }
    const unsigned lds0 = lds_address(lds), stat0 = lds_address(&lstat[0][0][0]);
    const float *stat = a.stats + ((long)b * a.Hkv + h) * a.stat_rows;
    // -> true: exactly PIECES instructions are on their way (and one more of waves 0 and 1)
    auto stage = [&](int it, int buf) {
        const int blk = blk0 + 2 * it;
        if (VEC) {
            if (wave < 2) lds_dma_words(stat + wave * a.stat_stride + blk * 32, lane, stat0 + buf * 512 + wave * 256);
            const bool p = sq.dma(lds0 + buf * 2 * TILE, blk, nq, rb, wave, lane);
            return sg.dma(lds0 + buf * 2 * TILE + TILE, blk, nq, rb, wave, lane) && p;
        }
        if (tid < 128) lstat[buf][wave][lane] = stat[wave * a.stat_stride + blk * 32 + lane];
        sq.copy(lds + buf * 2 * TILE, blk, nq, rb, a.vec, wave, lane);
        sg.copy(lds + buf * 2 * TILE + TILE, blk, nq, rb, a.vec, wave, lane);
        return false;
    };
    // bit i: the stage issued i stages ago is exactly PIECES instructions
    unsigned exact = 0;
    auto issue = [&](int it) {
        if (it < it1) exact = exact << 1 | (stage(it, (it - it0) % NBUF) ? 1u : 0u);
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) issue(it0 + i);

    typename Ops<T>::Frag kf[STEPS], vf[DK ? STEPS : 1];
    load_row<T, DP>(kf, row_at(a.k, b, j, h, sizeof(T)), a.Dk, j < nk, a.vec, lane);
    if (DK) load_row<T, DP>(vf, row_at(a.v, b, j, h, sizeof(T)), a.Dv, j < nk, a.vec, lane);
    f32x16 dk[DK ? DP / 32 : 1], dv[DV ? DP / 32 : 1];
    LaneMap<T, DP> map;
    map.init(lane);
    auto zero = [&] {
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                if (DK) dk[d][i] = 0.f;
                if (DV) dv[d][i] = 0.f;
            }
    };
    auto sees = [&](int r0) {
        const int at = r0 + 4 * (opaque(lane) >> 5);
        return Sees{by.hi - at, by.lo - at, -1};
    };
    zero();
    bool odd = false;                                    // a block with masked pairs holds values that are no numbers
    auto arrive = [&](int it) {
        if (NBUF == 1) {
            __syncthreads();
            stage(it, 0);
        }
        // the stages behind this one may still be on their way
        const int behind = min(AHEAD - 1, it1 - 1 - it);
        const bool counted = AHEAD > 1 && behind > 0 && (exact & ((1u << behind) - 1)) == (1u << behind) - 1;
        if (AHEAD > 1 && counted && behind == 1) dma_wait_but<PIECES>();
        else if (AHEAD > 2 && counted && behind == 2) dma_wait_but<2 * PIECES>();
        else dma_wait();
        __syncthreads();
        if (NBUF > 1) issue(it + AHEAD);
    };
    auto first_row = [&](int it) { return (blk0 + 2 * it + phase) * 32; };
    auto whole = [&](int it) { return first_row(it) >= full.lo && first_row(it) + 32 <= full.hi; };
    auto tile_of = [&](int it) { return lds0 + (it - it0) % NBUF * 2 * TILE + phase * 32 * TL::kRowBytes; };
    auto stats_of = [&](int it) { return RowStats{stat0 + (it - it0) % NBUF * 512 + phase * 128 + (lane >> 5) * 16}; };
    int it = it0;
    while (it < it1) {                                    // (two loops: see the rows kernel)
#pragma unroll 1
        for (; it < it1 && !whole(it); ++it) {
            arrive(it);
            if (idle) continue;
            const unsigned tq = tile_of(it), tg = tq + TILE;
            if (DV) odd = odd || block_not_finite<T, DP>(tg, 0, lane);
            if (DK) odd = odd || block_not_finite<T, DP>(tq, 0, lane);
            GradBlock<T, DP, DV, DK, true, RowStats> blk;
            blk.run(dk, dv, kf, vf, tq, tg, map, stats_of(it), sees(first_row(it)), a.scale_log2);
        }
#pragma unroll 1
        for (; it < it1 && whole(it); ++it) {
            arrive(it);
            const unsigned tq = tile_of(it), tg = tq + TILE;
            GradBlock<T, DP, DV, DK, false, RowStats> blk;
            blk.run(dk, dv, kf, vf, tq, tg, map, stats_of(it), Sees{}, a.scale_log2);
        }
    }
    if (__syncthreads_or(odd)) {                          // then the workgroup does its keys once more, with guarded products
        zero();
#pragma unroll 1
        for (it = it0; it < it1; ++it) {
            __syncthreads();
            stage(it, 0);
            dma_wait();
            __syncthreads();
            const int r0 = first_row(it);
            const unsigned tq = lds0 + phase * 32 * TL::kRowBytes, tg = tq + TILE;
            const RowStats stats = {stat0 + phase * 128 + (lane >> 5) * 16};
            GradBlock<T, DP, DV, DK, true, RowStats> blk;
            if (!idle) blk.run_guarded(dk, dv, kf, vf, tq, tg, map, stats, sees(r0), a.scale_log2, lane);
        }
    }
    // the odd blocks' sums join the even ones'
    float *sum = reinterpret_cast<float *>(lds) + (wave & 1) * DP * 32 + lane;
    auto join = [&](f32x16 *acc) {
        __syncthreads();
        if (phase == 1) {
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) sum[(d * 16 + i) * 64] = acc[d][i];
        }
        __syncthreads();
        if (phase == 0) {
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[d][i] += sum[(d * 16 + i) * 64];
        }
    };
    if constexpr (DK) join(dk);
    if constexpr (DV) join(dv);
    if (phase == 1 || j >= a.Tk) return;
    float *part = nullptr;
    const int slots = block_slots(a, block);
    if (slots > 1) {
        const long slot = slots_before(a, block) + (tail ? a.chunks + chunk : chunk);
        part = a.part + ((((long)b * a.Hkv + h) * slots_before(a, blocks) + slot) * kBwdKeys + (j - k0)) * (a.Dk + a.Dv);
    }
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int col = d * 32 + 8 * i + 4 * (lane >> 5);
            f32x4 v;
            if constexpr (DK) {
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = dk[d][4 * i + k] * a.scale;
                if (part) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (col + k < a.Dk) part[col + k] = v[k];
                } else store_grad<T>(a.dk, b, j, h, col, a.Dk, a.vec_out, v);
            }
            if constexpr (DV) {
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = dv[d][4 * i + k];
                if (part) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (col + k < a.Dv) part[a.Dk + col + k] = v[k];
                } else store_grad<T>(a.dv, b, j, h, col, a.Dv, a.vec_out, v);
            }
        }
}

// the slots of key blocks become their gradients, added in their order: four keys to a workgroup.  (8 sink blocks of 13 slots: 6 us; one load
// at a time 17.)
template <typename T>
__global__ __launch_bounds__(kHeadsThreads) void backward_join_kernel(BackwardArgs a, int blocks, int joined) {
    const int w = a.Dk + a.Dv;
    int id = blockIdx.x;
    const int quad = id % (kBwdKeys / 4);
    id /= kBwdKeys / 4;
    const int block = id % joined;
    id /= joined;
    const int h = id % a.Hkv, b = id / a.Hkv, key = quad * 4 + (threadIdx.x >> 6), j = block * kBwdKeys + key, slots = block_slots(a, block);
    if (j >= a.Tk) return;
    const float *src = a.part + ((((long)b * a.Hkv + h) * slots_before(a, blocks) + slots_before(a, block)) * kBwdKeys + key) * w;
    for (int c = threadIdx.x & 63; c < w; c += 64) {
        float sum = 0.f;
        for (int x0 = 0; x0 < slots; x0 += 8) {          // (eight loads on their way)
            float v[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) v[x] = x0 + x < slots ? src[(long)(x0 + x) * kBwdKeys * w + c] : 0.f;
#pragma unroll
            for (int x = 0; x < 8; ++x) sum += v[x];
        }
        T *row = c < a.Dk ? (T *)row_at(a.dk, b, j, h, sizeof(T)) + c : (T *)row_at(a.dv, b, j, h, sizeof(T)) + (c - a.Dk);
        *row = from_f32<T>(sum);
    }
}

// ---- the weights of every key: 32 KW keys to a workgroup --------------------------------------------------------------------------
// w_out_j = w_in_j + sum_i exp(s_ij - lse_i): the first half of the dK / dV walk, with column sums in place of the products.  KW waves lie
// along the keys, 4 / KW take the row blocks in turn; fragments come straight from memory (Q stays in the L2), no barriers in the loop.
template <typename T, int DP, int KW>
__global__ __launch_bounds__(kHeadsThreads) void weights_kernel(WeightArgs a, int G, int blocks) {
    constexpr int STEPS = DP / Ops<T>::kStep, PHASES = 4 / KW;
    __shared__ float part[4][32];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int id = xcd_place(blockIdx.x, gridDim.x);
    const int k0 = (id % blocks) * 32 * KW, j = k0 + wave % KW * 32 + (lane & 31);
    id /= blocks;
    const int h = id % a.Hkv, b = id / a.Hkv;
    const int nq = clamp_len(a.q_lens, b, a.Tq), nk = clamp_len(a.kv_lens, b, a.Tk);
    const SeenBy tok = seen_by(j, nq, nk, 1 << 30, 0), by = {tok.lo * G, tok.hi * G};
    float sum = 0.f;
    if (k0 < nk && nq > 0) {                             // (a call without queries may come without keys: nothing is read)
        typename Ops<T>::Frag kf[STEPS];
        load_row<T, DP>(kf, row_at(a.k, b, j, h, sizeof(T)), a.Dk, j < nk, a.vec, lane);
        const int r_end = nq * G, first = max(0, k0 - (nk - nq)) * G / 32 + wave / KW;
        for (int r0 = first * 32; r0 < r_end; r0 += 32 * PHASES) {
            const int r = r0 + (lane & 31), t = r / G, hq = h * G + r - t * G;
            typename Ops<T>::Frag qf[STEPS];
            load_row<T, DP>(qf, row_at(a.q, b, t, hq, sizeof(T)), a.Dk, r < r_end, a.vec, lane);
            const float lse2 = r < r_end ? a.lse[((long)b * a.Hq + hq) * a.Tq + t] * kLog2e : 0.f;
            f32x16 s = {};
#pragma unroll
            for (int i = 0; i < STEPS; ++i)
                if (sizeof(T) == 2 || i * Ops<T>::kStep < a.Dk) s = Ops<T>::mma(qf[i], kf[i], s);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int at = row_of(i, lane >> 5);
                const float ref = __shfl(lse2, at);
                if (r0 + at >= by.lo && r0 + at < by.hi) sum += __builtin_amdgcn_exp2f(s[i] * a.scale_log2 - ref);
            }
        }
    }
    sum = half_sum(sum);
    if (PHASES > 1) {
        if (lane < 32) part[wave][lane] = sum;
        __syncthreads();
        if (wave >= KW) return;
#pragma unroll
        for (int p = 1; p < PHASES; ++p) sum += part[wave + p * KW][lane & 31];
    }
    if (lane < 32 && j < a.Tk) {
        const float w = a.w_in[b * a.wi_batch + h * a.wi_head + j];
        a.w_out[b * a.wo_batch + h * a.wo_head + j] = w + sum;
    }
}

template <typename T, int DP, bool VEC>
void backward(const BackwardArgs &a, hipStream_t s) {
    constexpr int BN = DP * (int)sizeof(T) <= 256 ? 64 : 32;
    const int G = a.Hq / a.Hkv, rows = a.Tq * G, groups = a.B * a.Hkv, tiles = (rows + 127) / 128;
    if (tiles > 0) backward_rows_kernel<T, DP, BN, VEC><<<groups * tiles, kHeadsThreads, 0, s>>>(a, rows, G, tiles);
    const int blocks = (a.Tk + kBwdKeys - 1) / kBwdKeys, grid = groups * (blocks * a.chunks + a.sink_blocks * a.tail_chunks);
    if (blocks == 0) return;
    if constexpr (DP > 128) {
        backward_keys_kernel<T, DP, 1, VEC><<<grid, kHeadsThreads, 0, s>>>(a, G, blocks);
        backward_keys_kernel<T, DP, 2, VEC><<<grid, kHeadsThreads, 0, s>>>(a, G, blocks);
    } else {
        backward_keys_kernel<T, DP, 3, VEC><<<grid, kHeadsThreads, 0, s>>>(a, G, blocks);
    }
    const int joined = a.chunks > 1 ? blocks : a.tail_chunks > 0 ? a.sink_blocks : 0;
    if (joined > 0) backward_join_kernel<T><<<groups * joined * (kBwdKeys / 4), kHeadsThreads, 0, s>>>(a, blocks, joined);
}
template <typename T, int DP>
void backward(const BackwardArgs &a, hipStream_t s) {
    if (a.dma) backward<T, DP, true>(a, s);
    else backward<T, DP, false>(a, s);
}

template <typename T, int DP>
void weights(const WeightArgs &a, hipStream_t s) {
    if (a.Tk == 0) return;
    // 128 keys to a workgroup read Q a quarter as often; while they do not fill the chip the rows are split instead
    const int G = a.Hq / a.Hkv, wide = (a.Tk + 127) / 128, narrow = (a.Tk + 31) / 32;
    if ((long)a.B * a.Hkv * wide >= 512) weights_kernel<T, DP, 4><<<a.B * a.Hkv * wide, kHeadsThreads, 0, s>>>(a, G, wide);
    else weights_kernel<T, DP, 1><<<a.B * a.Hkv * narrow, kHeadsThreads, 0, s>>>(a, G, narrow);
}

}  // namespace
}  // namespace heads

hipError_t launch_attend_backward(const BackwardArgs &a, int dtype, hipStream_t s) {
    const int pad = heads_pad(a.Dk, a.Dv);
    if (dtype == SDPA_BF16) {
        if (pad == 64) heads::backward<__bf16, 64>(a, s);
        else if (pad == 128) heads::backward<__bf16, 128>(a, s);
        else heads::backward<__bf16, 256>(a, s);
    } else {
        if (pad == 64) heads::backward<float, 64>(a, s);
        else if (pad == 128) heads::backward<float, 128>(a, s);
        else heads::backward<float, 256>(a, s);
    }
    return hipGetLastError();
}

hipError_t launch_weights(const WeightArgs &a, int dtype, hipStream_t s) {
    const int pad = heads_pad(a.Dk, a.Dk);
    if (dtype == SDPA_BF16) {
        if (pad == 64) heads::weights<__bf16, 64>(a, s);
        else if (pad == 128) heads::weights<__bf16, 128>(a, s);
        else heads::weights<__bf16, 256>(a, s);
    } else {
        if (pad == 64) heads::weights<float, 64>(a, s);
        else if (pad == 128) heads::weights<float, 128>(a, s);
        else heads::weights<float, 256>(a, s);
    }
    return hipGetLastError();
}

}  // namespace sdpa
