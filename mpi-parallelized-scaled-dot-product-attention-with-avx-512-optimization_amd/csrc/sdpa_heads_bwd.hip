// sdpa_heads_bwd.hip -- gradients of attention_window, and the weights every key was given (attention_scored).
//
//     P = exp(s - lse) on visible pairs, dP = dO V^T, delta_i = sum_d dO_id O_id, dS = P * (dP - delta)
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

// ---- dQ: 128 rows to a workgroup, 32 to a wave -------------------------------------------------------------------------
// One 32-key block: S^T and dP^T with the keys as rows, dS^T kept in registers as the operand of dQ^T += K^T dS^T.
template <typename T, int DP, bool MASKED>
__device__ inline void grad_rows(f32x16 *dq, const typename Ops<T>::Frag *q, const typename Ops<T>::Frag *g, unsigned tk, unsigned tv,
                                 const LaneMap<T, DP> &map, int j0, Seen seen, int sinks, float scale, float lse2, float delta, int lane) {
    constexpr int STEPS = DP / Ops<T>::kStep;
    f32x16 s = {}, dp = {};
    const unsigned ak = tk + map.rows, av = tv + map.rows;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) s = Ops<T>::mma(read_rows<T, DP>(ak, 0, i), q[i], s);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) dp = Ops<T>::mma(read_rows<T, DP>(av, 0, i), g[i], dp);
    uint32_t vis = 0;
    const int half = MASKED ? opaque(lane) >> 5 : 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float p = __builtin_amdgcn_exp2f(s[i] * scale - lse2);
        s[i] = p * (dp[i] - delta);
        if (MASKED) {
            const int j = j0 + row_of(i, half);
            const bool ok = j < seen.hi && (j >= seen.lo || j < sinks);
            vis |= ok ? 1u << i : 0u;
            s[i] = ok ? s[i] : 0.f;
        }
    }
    mma_block<T, DP, DP / 32>(dq, tk, map, 0, to_probs(s, T()), MASKED, vis, 1, lane);
}

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
    float delta = 0.f;
    {
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
    const long at = ((long)b * a.Hq + hq) * a.Tq + t;
    const float lse2 = live ? a.lse[at] * kLog2e : 0.f;
    if (r < rows && lane < 32) a.delta[at] = delta;

    f32x16 dq[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) dq[d][i] = 0.f;
    LaneMap<T, DP> map;
    map.init(lane);
    for (int it = 0, buf = 0; it < count; ++it, buf ^= 1) {
        dma_wait();
        __syncthreads();
        if (it + 1 < count) stage(it + 1, buf ^ 1);
#pragma unroll 1
        for (int n = 0; n < BN / 32; ++n) {
            const Frame f = list.frame(it * BN + n * 32, 32);
            if (!sees_some(wv, f, 32)) continue;
            const unsigned tk = lds0 + buf * 2 * TILE + n * 32 * TL::kRowBytes, tv = tk + TILE;
            if (sees_all(wv, f, 32)) grad_rows<T, DP, false>(dq, q, g, tk, tv, map, f.j0, seen, f.sinks, a.scale_log2, lse2, delta, lane);
            else grad_rows<T, DP, true>(dq, q, g, tk, tv, map, f.j0, seen, f.sinks, a.scale_log2, lse2, delta, lane);
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
    // (groups of at most 32 heads) rows behind the last query are read as the last query's: their weights are masked
    __device__ void dma(unsigned lds, int block, int nq, const RowBlocks &rb, int wave, int lane) const {
        const int t0 = block * rb.tokens;
        const char *at = base + (long)t0 * token;
        const bool plain = dim == DP && rb.tokens * rb.G == 32, inside = t0 + 2 * rb.tokens <= nq;
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
            unsigned o = off[k];
            const unsigned dst = lds + (unsigned)(wave * kPieces + k) * 1024u;
            if (plain && inside) { lds_dma(at, o, dst); continue; }
            const int ln = opaque(lane), r = row(wave, ln, k), i = r & 31, t = t0 + (r >> 5) * rb.tokens + i / rb.G;
            if (t >= nq) o += (unsigned)((nq - 1 - t) * (int)token);
            if (i < rb.tokens * rb.G && source(wave, ln, k) * Ops<T>::kVec < dim) lds_dma(at, o, dst);     // (the rest stays zero)
        }
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

// One block of 32 rows against a wave's 32 keys: P, dP, dS have the rows as rows and a key to a lane, and stay in registers as the
// operands of dV^T += dO^T P and dK^T += Q^T dS.
template <typename T, int DP, int WHAT, bool MASKED>
__device__ inline void grad_keys(f32x16 *dk, f32x16 *dv, const typename Ops<T>::Frag *kf, const typename Ops<T>::Frag *vf, unsigned tq,
                                 unsigned tg, const LaneMap<T, DP> &map, unsigned stats, int r0, SeenBy by, float scale, int lane) {
    constexpr int STEPS = DP / Ops<T>::kStep;
    const unsigned aq = tq + map.rows, ag = tg + map.rows, st = stats + (lane >> 5) * 16;
    f32x16 s = {};
#pragma unroll
    for (int i = 0; i < STEPS; ++i) s = Ops<T>::mma(read_rows<T, DP>(aq, 0, i), kf[i], s);
    uint32_t vis = 0;
    const int half = MASKED ? opaque(lane) >> 5 : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f32x4 lse2 = lds_read<f32x4>(st, i * 32);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int x = 4 * i + k;
            s[x] = __builtin_amdgcn_exp2f(s[x] * scale - lse2[k]);
            if (MASKED) {
                const int r = r0 + row_of(x, half);
                const bool ok = r >= by.lo && r < by.hi;
                vis |= ok ? 1u << x : 0u;
                s[x] = ok ? s[x] : 0.f;
            }
        }
    }
    if constexpr ((WHAT & 1) != 0) mma_block<T, DP, DP / 32>(dv, tg, map, 0, to_probs(s, T()), MASKED, vis, 1, lane);
    if constexpr ((WHAT & 2) != 0) {
        f32x16 dp = {};
#pragma unroll
        for (int i = 0; i < STEPS; ++i) dp = Ops<T>::mma(read_rows<T, DP>(ag, 0, i), vf[i], dp);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4 delta = lds_read<f32x4>(st, 256 + i * 32);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int x = 4 * i + k;
                const float ds = s[x] * (dp[x] - delta[k]);
                s[x] = MASKED && !((vis >> x) & 1) ? 0.f : ds;
            }
        }
        mma_block<T, DP, DP / 32>(dk, tq, map, 0, to_probs(s, T()), MASKED, vis, 1, lane);
    }
}

// ---- dK, dV: 64 keys to a workgroup -----------------------------------------------------------------------------------------
// Waves 0 and 1 take 32 keys each on the even row blocks, waves 2 and 3 the same keys on the odd ones; the two sums are added in LDS
// at the end.  (Against four waves of 32 keys: twice the workgroups, so that two share a CU and one's exponentials run beside the
// other's products, for a second reading of Q and dO out of L2.)
// WHAT: 3 = both; heads of 256 do them one after the other (1 = dV, 2 = dK): two accumulators and two operands of 256 columns leave
// no registers for the scores.
template <typename T, int DP, int WHAT, bool VEC>
__global__ __launch_bounds__(kHeadsThreads, DP * (int)sizeof(T) <= 128 ? 2 : 1)
void backward_keys_kernel(BackwardArgs a, int G, int items) {
    using TL = Tile<T, DP>;
    constexpr int STEPS = DP / Ops<T>::kStep, TILE = 64 * TL::kRowBytes, NBUF = 4 * TILE <= 131072 ? 2 : 1;
    constexpr bool DV = (WHAT & 1) != 0, DK = (WHAT & 2) != 0;
    __shared__ __attribute__((aligned(1024))) char lds[2 * TILE * NBUF];     // Q, dO, Q, dO
    __shared__ __attribute__((aligned(16))) float lstat[2][2][64];            // [buffer][lse, delta][row]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int id = xcd_place(blockIdx.x, gridDim.x);
    const int item = id % items;
    id /= items;
    const int h = id % a.Hkv, b = id / a.Hkv;
    const int sink_items = a.sink_blocks * a.sink_chunks;
    const int chunks = item < sink_items ? a.sink_chunks : a.rest_chunks;
    const int block = item < sink_items ? item / chunks : a.sink_blocks + (item - sink_items) / chunks;
    const int chunk = item < sink_items ? item % chunks : (item - sink_items) % chunks;
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
    const int it0 = (int)((long)pairs * chunk / chunks), it1 = (int)((long)pairs * (chunk + 1) / chunks);

    RowStager<T, DP> sq, sg;
    sq.init(row_at(a.q, b, 0, h * G, sizeof(T)), a.q, a.Dk, rb, wave, lane);
    sg.init(row_at(a.dout, b, 0, h * G, sizeof(T)), a.dout, a.Dv, rb, wave, lane);
    if (VEC && (a.Dk < DP || a.Dv < DP || rb.tokens * G < 32)) {
        zero_lds(lds, 2 * TILE * NBUF, kHeadsThreads);
        __syncthreads();
    }
    const unsigned lds0 = lds_address(lds), stat0 = lds_address(&lstat[0][0][0]);
    float rl = 0.f, rd = 0.f;
    auto stage = [&](int it, int buf) {
        const int blk = blk0 + 2 * it;
        if (VEC) {
            sq.dma(lds0 + buf * 2 * TILE, blk, nq, rb, wave, lane);
            sg.dma(lds0 + buf * 2 * TILE + TILE, blk, nq, rb, wave, lane);
        } else {
            sq.copy(lds + buf * 2 * TILE, blk, nq, rb, a.vec, wave, lane);
            sg.copy(lds + buf * 2 * TILE + TILE, blk, nq, rb, a.vec, wave, lane);
        }
        if (tid < 64) {                                  // a row that does not exist: weight 2^(0 - inf) = 0
            const int i = tid & 31, bl = blk + (tid >> 5), t = rb.token(bl, i);
            const bool live = t < nq && rb.used(bl, i);
            const long at = ((long)b * a.Hq + h * G + rb.head(bl, i)) * a.Tq + t;
            rl = live ? a.lse[at] * kLog2e : __builtin_inff();
            rd = live ? a.delta[at] : 0.f;
        }
    };
    auto put_stat = [&](int buf) {
        if (tid < 64) { lstat[buf][0][tid] = rl; lstat[buf][1][tid] = rd; }
    };
    if (NBUF == 2 && it0 < it1) { stage(it0, 0); put_stat(0); }

    typename Ops<T>::Frag kf[STEPS], vf[DK ? STEPS : 1];
    load_row<T, DP>(kf, row_at(a.k, b, j, h, sizeof(T)), a.Dk, j < nk, a.vec, lane);
    if (DK) load_row<T, DP>(vf, row_at(a.v, b, j, h, sizeof(T)), a.Dv, j < nk, a.vec, lane);
    f32x16 dk[DK ? DP / 32 : 1], dv[DV ? DP / 32 : 1];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (DK) dk[d][i] = 0.f;
            if (DV) dv[d][i] = 0.f;
        }
    LaneMap<T, DP> map;
    map.init(lane);
    for (int it = it0, buf = 0; it < it1; ++it) {
        if (NBUF == 1) {
            __syncthreads();
            stage(it, 0);
            put_stat(0);
        }
        dma_wait();
        __syncthreads();
        if (NBUF == 2 && it + 1 < it1) stage(it + 1, buf ^ 1);
        const int r0 = (blk0 + 2 * it + phase) * 32;
        const unsigned tq = lds0 + buf * 2 * TILE + phase * 32 * TL::kRowBytes, tg = tq + TILE;
        const unsigned stats = stat0 + buf * 512 + phase * 128;
        if (r0 >= full.lo && r0 + 32 <= full.hi)
            grad_keys<T, DP, WHAT, false>(dk, dv, kf, vf, tq, tg, map, stats, r0, by, a.scale_log2, lane);
        else
            grad_keys<T, DP, WHAT, true>(dk, dv, kf, vf, tq, tg, map, stats, r0, by, a.scale_log2, lane);
        if (NBUF == 2) {
            buf ^= 1;
            if (it + 1 < it1) put_stat(buf);
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
    if (chunks > 1) {
        // partial rows lie item by item: first the sink blocks' (if they are shared), then the rest's
        const long base = a.sink_chunks > 1 ? 0 : sink_items;
        const long per = items - base - (a.rest_chunks > 1 ? 0 : items - sink_items);
        part = a.part + ((((long)b * a.Hkv + h) * per + (item - base)) * kBwdKeys + (j - k0)) * (a.Dk + a.Dv);
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

// the chunks of key blocks become their gradients, added in their order: four keys to a workgroup
template <typename T>
__global__ __launch_bounds__(kHeadsThreads) void backward_join_kernel(BackwardArgs a, int block0, int blocks, long item0, int chunks,
                                                                      long per) {
    const int w = a.Dk + a.Dv;
    int id = blockIdx.x;
    const int quad = id % (kBwdKeys / 4);
    id /= kBwdKeys / 4;
    const int blk = id % blocks;
    id /= blocks;
    const int h = id % a.Hkv, b = id / a.Hkv, key = quad * 4 + (threadIdx.x >> 6), j = (block0 + blk) * kBwdKeys + key;
    if (j >= a.Tk) return;
    const float *src = a.part + ((((long)b * a.Hkv + h) * per + item0 + (long)blk * chunks) * kBwdKeys + key) * w;
    for (int c = threadIdx.x & 63; c < w; c += 64) {
        float sum = 0.f;
        for (int x = 0; x < chunks; ++x) sum += src[(long)x * kBwdKeys * w + c];
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
    if (k0 < nk) {
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
    const int blocks = (a.Tk + kBwdKeys - 1) / kBwdKeys, rest = blocks - a.sink_blocks;
    const int sink_items = a.sink_blocks * a.sink_chunks, items = sink_items + rest * a.rest_chunks;
    if (items == 0) return;
    if constexpr (DP > 128) {
        backward_keys_kernel<T, DP, 1, VEC><<<groups * items, kHeadsThreads, 0, s>>>(a, G, items);
        backward_keys_kernel<T, DP, 2, VEC><<<groups * items, kHeadsThreads, 0, s>>>(a, G, items);
    } else {
        backward_keys_kernel<T, DP, 3, VEC><<<groups * items, kHeadsThreads, 0, s>>>(a, G, items);
    }
    const long base = a.sink_chunks > 1 ? 0 : sink_items, per = items - base - (a.rest_chunks > 1 ? 0 : items - sink_items);
    constexpr int quads = kBwdKeys / 4;
    if (a.sink_chunks > 1 && a.sink_blocks > 0)
        backward_join_kernel<T><<<groups * a.sink_blocks * quads, kHeadsThreads, 0, s>>>(a, 0, a.sink_blocks, 0, a.sink_chunks, per);
    if (a.rest_chunks > 1 && rest > 0)
        backward_join_kernel<T><<<groups * rest * quads, kHeadsThreads, 0, s>>>(a, a.sink_blocks, rest, sink_items - base, a.rest_chunks, per);
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
