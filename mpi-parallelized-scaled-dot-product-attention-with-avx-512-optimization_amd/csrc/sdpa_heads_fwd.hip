// sdpa_heads_fwd.hip -- attention of grouped heads over a cache: the kernels behind attention_window, attention_prefix and
// attention_scored.
//
// For a query row i with visible keys j:  s_ij = scale * q_i . k_j,  lse_i = log sum_j exp(s_ij),  out_i = sum_j
// exp(s_ij - lse_i) v_j.  One pass over the keys with a running maximum m and sum l (exp2 domain):
//     m' = max(m, max_j s_ij);  l' = l 2^(m-m') + sum_j 2^(s_ij - m');  O' = O 2^(m-m') + sum_j 2^(s_ij - m') v_j.
// The rows of a key head are its tokens' grouped heads, r = t * G + g, so that the G heads that share keys share the tile they
// are multiplied with, down to a single token.
#include "sdpa_heads_device.h"

namespace sdpa {
namespace heads {
namespace {

struct RowId { int b, t, g; bool live; };

__device__ inline RowId row_id(const AttendArgs &a, int b, int r, int rows, int G) {
    RowId x;
    const int bt = r / G;
    x.g = r - bt * G;
    if (a.shared) { x.b = bt / a.Tq; x.t = bt - x.b * a.Tq; }
    else { x.b = b; x.t = bt; }
    x.live = r < rows && x.t < (a.q_lens ? clamp_len(a.q_lens, x.b, a.Tq) : a.Tq);
    return x;
}

// what a lane keeps of its column: reference exponent, sum, the un-normalised row
template <int DP> struct State {
    float m, l;
    f32x16 o[DP / 32];
    __device__ void clear() {
        m = kNegInf; l = 0.f;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
    }
};

// ---- one tile of NB blocks of 32 keys against a wave's 32 rows, in three parts that a pipeline can take apart ------------------

// raw scores S^T = K Q^T
template <typename T, int DP, int NB>
__device__ inline void scores(f32x16 *s, const typename Ops<T>::Frag *q, unsigned lk, const LaneMap<T, DP> &map) {
    const unsigned at = lk + map.rows;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        s[n] = f32x16{};
#pragma unroll
        for (int i = 0; i < DP / Ops<T>::kStep; ++i)
            s[n] = Ops<T>::mma(read_rows<T, DP>(at, n, i), q[i], s[n]);
    }
}

// bit i: the lane's column sees row i of the block
__device__ inline uint32_t seen_bits(int j0, Seen seen, int sinks, int lane) {
    const int half = opaque(lane) >> 5;
    uint32_t vis = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int j = j0 + row_of(i, half);
        vis |= j < seen.hi && (j >= seen.lo || j < sinks) ? 1u << i : 0u;
    }
    return vis;
}
// what a lane's column does not see becomes -inf: the future, then what lies before the window (`low`: some of the tile may)
template <int NB> __device__ inline void hide(f32x16 *s, int j0, Seen seen, int sinks, bool low, int lane) {
    const int at = j0 + 4 * (opaque(lane) >> 5), hi = seen.hi - at, lo = seen.lo - at, sk = sinks - at;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[n][i] = n * 32 + row_of(i, 0) < hi ? s[n][i] : kNegInf;
    if (!low) return;
    if (j0 >= sinks) {
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[n][i] = n * 32 + row_of(i, 0) >= lo ? s[n][i] : kNegInf;
    } else {
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[n][i] = n * 32 + row_of(i, 0) >= lo || n * 32 + row_of(i, 0) < sk ? s[n][i] : kNegInf;
    }
}

// The reference exponent follows the maximum only when that rose by more than 2^8: a weight is then at most 2^8 instead of 1,
// which costs no precision (fp32 sums, and operand roundings are relative), and the 16 * DP / 32 multiplications of a rescale are
// rare.  The branch is the wave's, the decision each column's own: a row's bits must not depend on the rows beside it (a column
// without a row among them).  Scores are compared unscaled (the scale is positive: load_query) and scaled inside the exponential's
// argument.
// -> the exponent the tile's weights refer to
template <int NB> __device__ inline float largest(const f32x16 *s) {
    float mx = s[0][0];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = n == 0 ? 1 : 0; i < 16; ++i) mx = fmaxf(mx, s[n][i]);
    return mx;
}
template <int DP> __device__ inline float raise(State<DP> &st, float mx, float scale) {
    const float top = half_max(mx) * scale;
    const bool rises = top > st.m + 8.f;
    if (__any(rises)) {
        const float alpha = rises ? __builtin_amdgcn_exp2f(st.m - top) : 1.f;
        st.m = rises ? top : st.m;
        st.l *= alpha;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) st.o[d][i] *= alpha;
    }
    return st.m == kNegInf ? 0.f : st.m;                // (nothing seen yet: every weight is 2^-inf = 0)
}

// weights and their sum (the two lane halves' sums are joined once, behind the loop)
template <typename T, int DP, int NB>
__device__ inline void weigh(State<DP> &st, f32x16 *s, Probs<T> *p, float ref, float scale) {
    float sum = 0.f;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
#pragma unroll
        for (int i = 0; i < 16; ++i) { s[n][i] = __builtin_amdgcn_exp2f(s[n][i] * scale - ref); sum += s[n][i]; }
        p[n] = to_probs(s[n], T());
    }
    st.l += sum;
}

// the lane's row of kept scores, at this tile
template <int NB> __device__ inline void keep_scores(float *keep, const f32x16 *s, int lane) {
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<f32x4 *>(keep + n * 32 + 8 * i + 4 * (lane >> 5)) = f32x4{s[n][4 * i], s[n][4 * i + 1], s[n][4 * i + 2], s[n][4 * i + 3]};
}

// a tile with masked pairs, guarded
template <typename T, int DP, int NB>
__device__ inline void attend_blocks(State<DP> &st, const typename Ops<T>::Frag *q, unsigned lk, unsigned lv, const LaneMap<T, DP> &map,
                                     int j0, Seen seen, int sinks, float scale, int lane) {
    f32x16 s[NB];
    scores<T, DP, NB>(s, q, lk, map);
    hide<NB>(s, j0, seen, sinks, true, lane);
    const float ref = raise<DP>(st, largest<NB>(s), scale);
    Probs<T> p[NB];
    weigh<T, DP, NB>(st, s, p, ref, scale);
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        if (__builtin_expect(block_not_finite<T, DP>(lv, n, lane), 0))
            mma_block_guarded<T, DP, DP / 32>(st.o, lv, map, n, p[n], seen_bits(j0 + n * 32, seen, sinks, lane), 3);
        else
            mma_block<T, DP, DP / 32>(st.o, lv, map, n, p[n], false, 0u, 3, lane);
    }
}

// An infinity that a row sees, times what is left of its weight (0, or of the other sign), has become NaN: then the guarded way, too.
template <typename T, int DP> __device__ inline bool lost_infinity(const State<DP> &st) {
    if (sizeof(T) == 4) return false;
    float bad = 0.f;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) bad = __builtin_fmaf(st.o[d][i], 0.f, bad);
    return __any(bad != bad);
}

// a finished row (or its partial triple): 4 consecutive values of row `x`, columns d .. d + 3
template <typename T>
__device__ inline void store4(const AttendArgs &a, const RowId &x, int hq, int d, f32x4 v) {
    T *row = (T *)a.out.data + x.b * a.out.batch + x.t * a.out.token + hq * a.out.head;
    if (a.vec_out) {
        if (d >= a.Dv) return;
        union { T e[4]; uint64_t u; f32x4 f; } y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y.e[i] = from_f32<T>(v[i]);
        if (sizeof(T) == 2) *reinterpret_cast<uint64_t *>(row + d) = y.u;
        else *reinterpret_cast<f32x4 *>(row + d) = y.f;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (d + i < a.Dv) row[d + i] = from_f32<T>(v[i]);
    }
}

__device__ inline void store_part4(const AttendArgs &a, long slot_row, int d, f32x4 v) {
    float *row = a.part + slot_row * a.Dv;
    if (a.Dv % 4 == 0) {
        if (d < a.Dv) *reinterpret_cast<f32x4 *>(row + d) = v;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (d + i < a.Dv) row[d + i] = v[i];
    }
}

// the statistics of a row: lse, or the slot's (m, l).  An empty row: out 0, lse -inf.
__device__ inline void store_stat(const AttendArgs &a, const RowId &x, int hq, int slot, float m, float l) {
    if (a.part) a.stat[((long)slot * a.B + x.b) * a.Tq * a.Hq + (long)x.t * a.Hq + hq] = make_float2(m, l);
    else a.lse[((long)x.b * a.Hq + hq) * a.Tq + x.t] = l == 0.f ? kNegInf : (m + __log2f(l)) * kLn2;
}

// A lane's column of Q.  The softmax scale is kept positive: a negative one turns the sign of the queries (exactly), and a scale of
// zero is queries of zero.
template <typename T, int DP>
__device__ inline void load_query(typename Ops<T>::Frag *q, const AttendArgs &a, const RowId &x, int hq, int lane) {
    const T *row = (const T *)a.q.data + x.b * a.q.batch + x.t * a.q.token + hq * a.q.head;
    const bool live = x.live && a.q_sign != 0;
    const uint32_t turn = a.q_sign < 0 ? (sizeof(T) == 2 ? 0x80008000u : 0x80000000u) : 0u;
#pragma unroll
    for (int s = 0; s < DP / Ops<T>::kStep; ++s) {
        union { u32x4 u; typename Ops<T>::Frag f; } y;
        y.u = u32x4{0, 0, 0, 0};
        if (live) y.u = load_chunk(row, s * Ops<T>::kStep + (lane >> 5) * Ops<T>::kVec, a.Dk, a.vec) ^ turn;
        q[s] = y.f;
    }
}

// ---- the steady state: scores of the next tile beside the weights of this one ---------------------------------------------------
// The tile's products are a list of units -- for each 32-key block the K units (a step of the next tile's scores), then the V units
// (a piece of O += V^T P) -- and a unit is written down as it is to be issued: the LDS read of the unit three ahead, this unit's
// matrix instructions, and a few of the vector instructions that are due.  hipcc left alone puts all exponentials first and every
// read right in front of its use (5000 cycles a tile and wave of 64 keys and 128 columns, against 1024 of its matrix instructions with
// weights in one term, 1536 in two).
template <typename T, int DP, int NB> struct Pipe {
    static constexpr int KU = DP / Ops<T>::kStep, VK = sizeof(T) == 2 ? 2 : 4, VU = DP / 32 * VK, PER = KU + VU, UNITS = NB * PER, AHEAD = 3;
    using Frag = typename Ops<T>::Frag;
    __device__ static Frag fetch(int u, unsigned ak, unsigned av) {
        const int n = u / PER, x = u % PER;
        if (x < KU) return read_rows<T, DP>(ak, n, x);
        return read_cols_part<DP>(av, n, (x - KU) / VK, (x - KU) % VK, T());
    }
    Frag ring[AHEAD + 1];
    Probs<T> p[NB];
    float sum, mx;
    template <int U>
    __device__ inline __attribute__((always_inline)) void unit(State<DP> &st, const Frag *q, f32x16 *s, f32x16 *s2, unsigned ak, unsigned av,
                                                               float ref, float scale) {
        if constexpr (U < UNITS) {
            constexpr int n = U / PER, x = U % PER;
            if constexpr (U + AHEAD < UNITS) ring[(U + AHEAD) % (AHEAD + 1)] = fetch(U + AHEAD, ak, av);
            const Frag f = ring[U % (AHEAD + 1)];
            if constexpr (x < KU) s2[n] = Ops<T>::mma(f, q[x], s2[n]);
            else st.o[(x - KU) / VK] = mma_part(f, p[n], (x - KU) % VK, st.o[(x - KU) / VK]);
            // weights: block 0's beside its K units, block m's between the V units of block m - 1 and its own
#pragma unroll
            for (int m = 0; m < NB; ++m) {
                const int first = m == 0 ? 0 : (m - 1) * PER + KU, count = m == 0 ? KU : PER;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (first + i * count / 16 == U) {
                        s[m][i] = __builtin_amdgcn_exp2f(s[m][i] * scale - ref);
                        sum += s[m][i];
                        if (sizeof(T) == 4 || (i & 1)) put_prob(p[m], s[m], i);
                    }
            }
            // the next tile's maximum, beside the last V units
            if constexpr (U >= UNITS - VU) {
#pragma unroll
                for (int i = 0; i < 16 * NB; ++i)
                    if (i * VU / (16 * NB) == U - (UNITS - VU)) mx = fmaxf(mx, s2[i / 16][i % 16]);
                asm volatile("" : "+v"(mx));             // (here, and not behind the last unit)
            }
            __builtin_amdgcn_sched_barrier(0);
            unit<U + 1>(st, q, s, s2, ak, av, ref, scale);
        }
    }
    // -> the maximum of the next tile's scores in s2
    __device__ inline __attribute__((always_inline)) float run(State<DP> &st, const Frag *q, f32x16 *s, f32x16 *s2, unsigned ak, unsigned av,
                                                               float ref, float scale) {
        sum = 0.f;
        mx = kNegInf;
#pragma unroll
        for (int n = 0; n < NB; ++n) s2[n] = f32x16{};
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) ring[u] = fetch(u, ak, av);
        __builtin_amdgcn_sched_barrier(0);
        unit<0>(st, q, s, s2, ak, av, ref, scale);
        st.l += sum;
        return mx;
    }
};

// ---- many rows: a workgroup's four waves share every key tile, each owns 32 rows -------------------------------------------------
// The loop is a pipeline over the tiles.  LDS holds two K tiles and two V tiles; K runs one tile ahead of V, the DMA one ahead of both,
// one barrier a tile.  A prompt of 8192 tokens, 32 heads on 8 of 128 columns, window 1024, bf16: 240 us, 129 GFLOP = 540 TFLOP/s.  Counters: a
// SIMD's matrix instructions (the weights are two operands) take 0.39 of its cycles, its vector instructions 0.40, and a wave waits 0.31 of
// its time: the two waves of a SIMD fill each other's pauses in part only.
template <typename T, int DP, int BN, bool VEC>
__global__ __launch_bounds__(kHeadsThreads, DP <= 128 ? 2 : 1)
void attend_rows_kernel(AttendArgs a, int rows, int G, int tiles) {
    using TL = Tile<T, DP>;
    constexpr int TILE = BN * TL::kRowBytes, NB = BN / 32, STEPS = DP / Ops<T>::kStep;
    __shared__ __attribute__((aligned(1024))) char lds[4 * TILE];            // K, K, V, V
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int id = xcd_place(blockIdx.x, gridDim.x);
    const int tile = tiles - 1 - id % tiles;             // (the rows that see most keys first)
    id /= tiles;
    const int split = id % a.splits;
    id /= a.splits;
    const int h = id % a.Hkv, b = id / a.Hkv;
    const int r0 = tile * 128, rw = r0 + wave * 32;
    const RowId x = row_id(a, b, rw + (lane & 31), rows, G);
    const int hq = h * G + x.g;

    SeenRange wg, wv;
    Seen seen = {0, 0};
    if (a.shared) {
        wg = SeenRange{a.Tk, a.Tk, 0, 0};
        wv = wg;
        if (x.live) seen.hi = a.Tk;
    } else {
        const int nq = clamp_len(a.q_lens, b, a.Tq), nk = clamp_len(a.kv_lens, b, a.Tk);
        wg = seen_range(r0 / G, min(r0 + 127, rows - 1) / G, nq, nk, a.window);
        wv = seen_range(rw / G, min(rw + 31, rows - 1) / G, nq, nk, a.window);
        if (x.live) seen = seen_at(nk - nq + x.t, nk, a.window);
    }
    const KeyList list = key_list(wg, a.sinks);
    const int count = list.tiles(BN), it0 = (int)((long)count * split / a.splits), it1 = (int)((long)count * (split + 1) / a.splits);
    Stager<T, DP, BN, 4> sk, sv;
    sk.init((const T *)a.k.data + (a.shared ? 0 : b * a.k.batch) + h * a.k.head, a.k.token, a.Dk, wave, lane);
    sv.init((const T *)a.v.data + (a.shared ? 0 : b * a.v.batch) + h * a.v.head, a.v.token, a.Dv, wave, lane);
    if (VEC && (a.Dk < DP || a.Dv < DP)) {
        zero_lds(lds, 4 * TILE, kHeadsThreads);
        __syncthreads();
    }
    const unsigned lds0 = lds_address(lds);
    auto stage_at = [&](const Stager<T, DP, BN, 4> &stager, int it, int place) {
        if (VEC) stager.dma(lds0 + place * TILE, it * BN, list, wave, lane);
        else stager.copy(lds + place * TILE, it * BN, list, wave, lane);
    };
    auto stage_k = [&](int it) { if (it < it1) stage_at(sk, it, (it - it0) & 1); };
    auto stage_v = [&](int it) { if (it < it1) stage_at(sv, it, 2 + ((it - it0) & 1)); };
    stage_k(it0);

    typename Ops<T>::Frag q[STEPS];
    load_query<T, DP>(q, a, x, hq, lane);
    State<DP> st;
    st.clear();
    LaneMap<T, DP> map;
    map.init(lane);
    f32x16 s[NB];
    float mx = kNegInf;
    bool cur = false, odd = false;                       // odd: a tile with masked pairs holds values that are no numbers
    if (it0 < it1) {
        dma_wait();
        __syncthreads();
        stage_k(it0 + 1);
        stage_v(it0);
        cur = sees_some(wv, list.frame(it0 * BN, BN), BN);
        if (cur) {
            scores<T, DP, NB>(s, q, lds0, map);
            mx = largest<NB>(s);
        }
    }
#pragma unroll 1
    for (int it = it0; it < it1; ++it) {
        const int buf = (it - it0) & 1;
        dma_wait();
        __syncthreads();
        stage_k(it + 2);
        stage_v(it + 1);
        const unsigned lk = lds0 + (buf ^ 1) * TILE, lv = lds0 + (2 + buf) * TILE;
        const bool had = cur;
        cur = it + 1 < it1 && sees_some(wv, list.frame((it + 1) * BN, BN), BN);
        if (!had) {
            if (cur) {
                scores<T, DP, NB>(s, q, lk, map);
                mx = largest<NB>(s);
            }
            continue;
        }
        const Frame f = list.frame(it * BN, BN);
        if (!sees_all(wv, f, BN)) {
            hide<NB>(s, f.j0, seen, f.sinks, f.j0 < wv.lo_max, lane);
            mx = largest<NB>(s);
#pragma unroll 1
            for (int n = 0; n < NB; ++n) odd = odd || block_not_finite<T, DP>(lv, n, lane);
        }
        const float ref = raise<DP>(st, mx, a.scale_log2);
        // (behind the last tile the scores of a stale tile are multiplied and dropped)
        f32x16 s2[NB];
        Pipe<T, DP, NB> pipe;
        mx = pipe.run(st, q, s, s2, lk + map.rows, lv + map.cols, ref, a.scale_log2);
#pragma unroll
        for (int n = 0; n < NB; ++n) s[n] = s2[n];
    }
    odd = odd || lost_infinity<T, DP>(st);
    // Such a tile gave NaN to rows that do not see it: the workgroup does its rows once more, with a guarded product and
    // otherwise the same arithmetic.
    if (__syncthreads_or(odd)) {
        st.clear();
#pragma unroll 1
        for (int it = it0; it < it1; ++it) {
            __syncthreads();
            stage_at(sk, it, 0);
            stage_at(sv, it, 2);
            dma_wait();
            __syncthreads();
            const Frame f = list.frame(it * BN, BN);
            if (sees_some(wv, f, BN))
                attend_blocks<T, DP, NB>(st, q, lds0, lds0 + 2 * TILE, map, f.j0, seen, f.sinks, a.scale_log2, lane);
        }
    }
    st.l = half_sum(st.l);
    if (!x.live) { st.m = kNegInf; st.l = 0.f; }         // (tiles that need no mask gave weights to rows that do not exist)
    if (rw + (lane & 31) >= rows) return;
    const int slot = a.slot0 + split;
    if (lane < 32) store_stat(a, x, hq, slot, st.m, st.l);
    const float inv = st.l == 0.f ? 0.f : 1.f / st.l;
    const long slot_row = ((long)slot * a.B + x.b) * a.Tq * a.Hq + (long)x.t * a.Hq + hq;
    if (a.part && st.l == 0.f) return;                   // (the join does not read an empty slot)
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int col = d * 32 + 8 * i + 4 * (lane >> 5);
            f32x4 v = {st.o[d][4 * i], st.o[d][4 * i + 1], st.o[d][4 * i + 2], st.o[d][4 * i + 3]};
            if (a.part) store_part4(a, slot_row, col, v);
            else {
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = st.l == 0.f ? 0.f : v[k] * inv;
                store4<T>(a, x, hq, col, v);
            }
        }
}

// ---- few rows (single tokens): the waves share 32 rows and take the key tiles in turn ------------------------------------
// Bound by the reading of the cache.  Every wave stages its own tiles of 32 keys (no barriers), the next one on its way by DMA while this
// one is multiplied: 64 KiB in flight on a CU.  (fp32 tiles are bound by their matrix instructions and are not double-buffered.)
// WIDE: up to eight waves, for calls so small that one workgroup does the keys of a head and no join is launched (one token of 16
// heads on 4 of 64 columns, a window of 512: 17.5 us with the call around it, 10.8 of them the kernel's four workgroups, which take their
// tiles one after the other; 21 us in two launches).
// Measured, 32 heads on 8 of 128 columns, bf16: 48 tokens over windows of 4096 160 us, 806 MB = 5.0 TB/s; 16 tokens over up to 8192 keys
// with their scores kept 89 us, 377 MB = 4.2 TB/s.
template <typename T, int DP, bool WIDE> struct FewShape {
    static constexpr int kPair = few_pair_bytes(DP, sizeof(T));                              // a K and a V tile
    static constexpr int kWaves = WIDE ? few_wide_waves(DP, sizeof(T)) : kPair * 8 <= 131072 || (sizeof(T) == 4 && DP == 128) ? 4 : 2;
    static constexpr int kBufs = (sizeof(T) == 2 || DP == 64) && kPair * 2 * kWaves <= 131072 ? 2 : 1;
};
template <typename T, int DP, bool WIDE, bool VEC>
__global__ __launch_bounds__((FewShape<T, DP, WIDE>::kWaves * 64)) void attend_few_kernel(AttendArgs a, int rows, int G) {
    using TL = Tile<T, DP>;
    constexpr int WAVES = FewShape<T, DP, WIDE>::kWaves, NBUF = FewShape<T, DP, WIDE>::kBufs;
    constexpr int TILE = 32 * TL::kRowBytes, WAVE_BYTES = 2 * TILE * NBUF;
    static_assert(WAVE_BYTES >= 32 * DP * 4, "the waves' rows are joined in the same memory");
    __shared__ __attribute__((aligned(1024))) char lds[WAVES * WAVE_BYTES];
    __shared__ float lm[WAVES][32], ll[WAVES][32];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int id = xcd_place(blockIdx.x, gridDim.x);
    const int split = id % a.splits;
    id /= a.splits;
    const int h = id % a.Hkv, b = id / a.Hkv;
    const RowId x = row_id(a, b, lane & 31, rows, G);
    const int hq = h * G + x.g;

    SeenRange wg;
    Seen seen = {0, 0};
    if (a.shared) {
        wg = SeenRange{a.Tk, a.Tk, 0, 0};
        if (x.live) seen.hi = a.Tk;
    } else {
        const int nq = clamp_len(a.q_lens, b, a.Tq), nk = clamp_len(a.kv_lens, b, a.Tk);
        wg = seen_range(0, a.Tq - 1, nq, nk, a.window);
        if (x.live) seen = seen_at(nk - nq + x.t, nk, a.window);
    }
    const KeyList list = key_list(wg, a.sinks);
    const int count = list.tiles(32), it0 = (int)((long)count * split / a.splits), it1 = (int)((long)count * (split + 1) / a.splits);

    char *mine = lds + wave * WAVE_BYTES;
    const unsigned lds0 = lds_address(mine);
    Stager<T, DP, 32, 1> sk, sv;
    sk.init((const T *)a.k.data + (a.shared ? 0 : b * a.k.batch) + h * a.k.head, a.k.token, a.Dk, 0, lane);
    sv.init((const T *)a.v.data + (a.shared ? 0 : b * a.v.batch) + h * a.v.head, a.v.token, a.Dv, 0, lane);
    if (VEC && (a.Dk < DP || a.Dv < DP)) {               // (its own part only: no barrier)
        for (int i = lane * 16; i < WAVE_BYTES; i += 1024) *reinterpret_cast<u32x4 *>(mine + i) = u32x4{0, 0, 0, 0};
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    // -> true: exactly 2 * kPieces instructions are on their way
    auto stage = [&](int it, int buf) {
        if (VEC) {
            const bool p = sk.dma(lds0 + buf * 2 * TILE, it * 32, list, 0, lane);
            return sv.dma(lds0 + buf * 2 * TILE + TILE, it * 32, list, 0, lane) && p;
        }
        sk.copy(mine + buf * 2 * TILE, it * 32, list, 0, lane);
        sv.copy(mine + buf * 2 * TILE + TILE, it * 32, list, 0, lane);
        return false;
    };
    if (NBUF == 2 && it0 + wave < it1) stage(it0 + wave, 0);
    typename Ops<T>::Frag q[DP / Ops<T>::kStep];
    load_query<T, DP>(q, a, x, hq, lane);
    State<DP> st;
    st.clear();
    LaneMap<T, DP> map;
    map.init(lane);
    // (kept scores: the row of a lane that has one; the list of attention_scored is the cache itself)
    float *kept = a.scores && (lane & 31) < rows ? a.scores + (((long)b * a.Hkv + h) * rows + (lane & 31)) * a.score_ld : nullptr;
    // One way through the products for masked tiles and others: a second one would have the accumulators in other registers (8 tokens against
    // 2048 keys, 8 heads on 2 of 256 columns: bf16 21 us, fp32 53; with a second way 1.37 and 1.11 times that).  fp32 heads of 256
    // columns still go through scratch memory, 58 accesses a tile.
    bool odd = false;                                    // a tile with masked pairs holds values that are no numbers
#pragma unroll 1
    for (int it = it0 + wave, buf = 0; it < it1; it += WAVES) {
        bool exact = false;
        if (NBUF == 1) stage(it, 0);
        else if (it + WAVES < it1) exact = stage(it + WAVES, buf ^ 1);
        if (NBUF == 2 && exact) dma_wait_but<2 * Stager<T, DP, 32, 1>::kPieces>();
        else dma_wait();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");       // (a wave reads only what it staged itself)
        const unsigned lk = lds0 + buf * 2 * TILE, lv = lk + TILE;
        const Frame f = list.frame(it * 32, 32);
        const bool masked = !sees_all(wg, f, 32);
        f32x16 s[1];
        scores<T, DP, 1>(s, q, lk, map);
        if (masked) {
            hide<1>(s, f.j0, seen, f.sinks, true, lane);
            odd = odd || block_not_finite<T, DP>(lv, 0, lane);
        }
        if (kept) keep_scores<1>(kept + it * 32, s, lane);
        const float ref = raise<DP>(st, largest<1>(s), a.scale_log2);
        Probs<T> p[1];
        weigh<T, DP, 1>(st, s, p, ref, a.scale_log2);
        mma_block<T, DP, DP / 32>(st.o, lv, map, 0, p[0], false, 0u, 3, lane);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");           // (its reads are over before the tile is written again)
        if (NBUF == 2) buf ^= 1;
    }
    odd = odd || lost_infinity<T, DP>(st);
    if (odd) {                                           // then the wave does its tiles once more, with guarded products
        st.clear();
#pragma unroll 1
        for (int it = it0 + wave; it < it1; it += WAVES) {
            stage(it, 0);
            dma_wait();
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            const Frame f = list.frame(it * 32, 32);
            attend_blocks<T, DP, 1>(st, q, lds0, lds0 + TILE, map, f.j0, seen, f.sinks, a.scale_log2, lane);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    }
    st.l = half_sum(st.l);
    if (!x.live) { st.m = kNegInf; st.l = 0.f; }         // (blocks that need no mask gave weights to rows that do not exist)
    // the waves' triples become one
    if (lane < 32) { lm[wave][lane] = st.m; ll[wave][lane] = st.l; }
    __syncthreads();
    const int col = lane & 31;
    float m = lm[0][col];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) m = fmaxf(m, lm[w][col]);
    const float ref = m == kNegInf ? 0.f : m;
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) l += ll[w][col] * __builtin_amdgcn_exp2f(lm[w][col] - ref);
    const float alpha = __builtin_amdgcn_exp2f(st.m - ref);
    float *lo = reinterpret_cast<float *>(mine);
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) lo[(d * 32 + row_of(i, lane >> 5)) * 32 + col] = st.l == 0.f ? 0.f : st.o[d][i] * alpha;
    __syncthreads();
    if (col >= rows) return;
    const int slot = a.slot0 + split;
    if (wave == 0 && lane < 32) store_stat(a, x, hq, slot, m, l);
    if (a.part && l == 0.f) return;
    const float inv = a.part ? 1.f : l == 0.f ? 0.f : 1.f / l;
    const long slot_row = ((long)slot * a.B + x.b) * a.Tq * a.Hq + (long)x.t * a.Hq + hq;
    constexpr int RUN = DP / (2 * WAVES);                // columns of a thread
    const int d0 = (tid >> 5) * RUN;
#pragma unroll
    for (int d = 0; d < RUN; d += 4) {
        f32x4 v = {};
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float *src = reinterpret_cast<const float *>(lds + w * WAVE_BYTES);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += src[(d0 + d + i) * 32 + col];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = l == 0.f ? 0.f : v[i] * inv;
        if (a.part) store_part4(a, slot_row, d0 + d, v);
        else store4<T>(a, x, hq, d0 + d, v);
    }
}

// ---- the join of the slots: the merge of partial triples ------------------------------------------------------------
// 32 lanes to a row's columns.  GROUPS = 8: a workgroup to a row, its eight groups of lanes to the slots in turn (2048 rows of 34 slots take
// 12 us, against 34 us with GROUPS = 1).  GROUPS = 1: eight rows to a workgroup (13986 rows of 5 slots: 7 us against 22 us).
template <typename T, int GROUPS>
__device__ inline void combine_row(const AttendArgs &a, int slots, long block) {
    __shared__ f32x4 sum[8][64];
    const long rows = (long)a.B * a.Tq * a.Hq;
    const int lane = threadIdx.x & 31, group = GROUPS == 8 ? threadIdx.x >> 5 : 0;
    const long r = GROUPS == 8 ? block : block * 8 + (threadIdx.x >> 5);
    if (GROUPS == 1 && r >= rows) return;
    float m = kNegInf;
    for (int s = 0; s < slots; s += 32) {
        float2 ml = make_float2(kNegInf, 0.f);
        if (s + lane < slots) ml = a.stat[(s + lane) * rows + r];
        m = fmaxf(m, ml.y != 0.f ? ml.x : kNegInf);
    }
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
    const float ref = m == kNegInf ? 0.f : m;
    float l = 0.f;
    for (int s = 0; s < slots; s += 32) {
        float2 ml = make_float2(kNegInf, 0.f);
        if (s + lane < slots) ml = a.stat[(s + lane) * rows + r];
        if (ml.y != 0.f) l += ml.y * __builtin_amdgcn_exp2f(ml.x - ref);
    }
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) l += __shfl_xor(l, d);
    f32x4 acc[2] = {};
    for (int s = group; s < slots; s += GROUPS) {
        const float2 ml = a.stat[s * rows + r];
        if (ml.y == 0.f) continue;                       // (an empty slot was not written)
        const float w = __builtin_amdgcn_exp2f(ml.x - ref);
        const float *src = a.part + (s * rows + r) * a.Dv;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int d = k * 128 + lane * 4;
            if (a.Dv % 4 == 0) {
                if (d < a.Dv) acc[k] += w * *reinterpret_cast<const f32x4 *>(src + d);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (d + i < a.Dv) acc[k][i] += w * src[d + i];
            }
        }
    }
    RowId x;
    const int hq = (int)(r % a.Hq);
    const long bt = r / a.Hq;
    x.b = (int)(bt / a.Tq); x.t = (int)(bt - (long)x.b * a.Tq); x.g = 0; x.live = true;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (lane == 0 && group == 0) a.lse[((long)x.b * a.Hq + hq) * a.Tq + x.t] = l == 0.f ? kNegInf : (m + __log2f(l)) * kLn2;
    if (GROUPS == 1) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (k * 128 + lane * 4 < a.Dv) store4<T>(a, x, hq, k * 128 + lane * 4, acc[k] * inv);
        return;
    }
    sum[group][lane] = acc[0];
    sum[group][32 + lane] = acc[1];
    __syncthreads();
    const int d = threadIdx.x * 4;
    if (d >= a.Dv) return;
    f32x4 v = sum[0][threadIdx.x];
#pragma unroll
    for (int g = 1; g < 8; ++g) v += sum[g][threadIdx.x];
    store4<T>(a, x, hq, d, v * inv);
}
template <typename T, int GROUPS>
__global__ __launch_bounds__(kHeadsThreads) void combine_kernel(AttendArgs a, int slots) { combine_row<T, GROUPS>(a, slots, blockIdx.x); }
// what the two ways measured above say: a workgroup to a row where its slots are many or the rows few
inline int combine_groups(long rows, int slots) { return slots > 8 || rows < 2048 ? 8 : 1; }
inline unsigned combine_blocks(long rows, int groups) { return (unsigned)(groups == 8 ? rows : (rows + 7) / 8); }

// w_out_j = w_in_j + sum over the rows of exp2(s_j - lse), from the kept scores: 1024 keys of a head to a workgroup
__device__ inline void add_weights(const WeightArgs &w, int block) {
    const int blocks = (w.Tk + 1023) / 1024, part = block % blocks, bh = block / blocks, h = bh % w.Hkv, b = bh / w.Hkv, G = w.Hq / w.Hkv;
    const int nq = clamp_len(w.q_lens, b, w.Tq), nk = clamp_len(w.kv_lens, b, w.Tk), rows = nq * G, all = w.Tq * G;
    __shared__ float lse2[kFewRows];
    __shared__ int last[kFewRows];                       // the last key a row sees
    if ((int)threadIdx.x < rows) {
        const int t = threadIdx.x / G, hq = h * G + threadIdx.x - t * G;
        float x;
        if (w.stat) {
            const long n = (long)w.B * w.Tq * w.Hq, r = ((long)b * w.Tq + t) * w.Hq + hq;
            float m = kNegInf, l = 0.f;
            for (int s = 0; s < w.slots; ++s) {
                const float2 ml = w.stat[s * n + r];
                if (ml.y == 0.f) continue;
                const float top = fmaxf(m, ml.x);
                l = l * __builtin_amdgcn_exp2f(m - top) + ml.y * __builtin_amdgcn_exp2f(ml.x - top);
                m = top;
            }
            x = l == 0.f ? kNegInf : m + __log2f(l);
        } else x = w.lse[((long)b * w.Hq + hq) * w.Tq + t] * kLog2e;
        last[threadIdx.x] = nk - nq + t;
        lse2[threadIdx.x] = x == kNegInf ? __builtin_inff() : x;         // (a row that sees nothing gives nothing)
    }
    __syncthreads();
    const int j = part * 1024 + threadIdx.x * 4;
    if (j >= w.Tk) return;
    f32x4 sum = {};
    if (j < nk) {
        const float *src = w.scores + (long)bh * all * w.score_ld + j;
#pragma unroll 4
        for (int r = 0; r < rows; ++r) {
            const f32x4 s = *reinterpret_cast<const f32x4 *>(src + (long)r * w.score_ld);
#pragma unroll
            for (int i = 0; i < 4; ++i)                  // (by the key's place: a row whose lse is no number gives nothing to what it does not see)
                sum[i] += j + i <= last[r] ? __builtin_amdgcn_exp2f(s[i] * w.scale_log2 - lse2[r]) : 0.f;
        }
    }
    const float *in = w.w_in + b * w.wi_batch + h * w.wi_head + j;
    float *out = w.w_out + b * w.wo_batch + h * w.wo_head + j;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (j + i < w.Tk) out[i] = in[i] + (j + i < nk ? sum[i] : 0.f);
}
template <typename T, int GROUPS>
__global__ __launch_bounds__(kHeadsThreads) void combine_scored_kernel(AttendArgs a, WeightArgs w, int slots, int blocks) {
    if ((int)blockIdx.x < blocks) combine_row<T, GROUPS>(a, slots, blockIdx.x);
    else add_weights(w, blockIdx.x - blocks);
}

template <typename T, int DP>
void attend(const AttendArgs &a, int rows, int G, int groups, hipStream_t s) {
    constexpr int BN = DP * (int)sizeof(T) <= 256 ? 64 : 32;
    if (rows <= kFewRows) {
        using Plain = FewShape<T, DP, false>;
        using Wide = FewShape<T, DP, true>;              // (fp32 above 64 columns: 128 KiB are the plain form's waves)
        constexpr int threads = Plain::kWaves * 64;
        constexpr bool WIDE = Wide::kWaves != Plain::kWaves || Wide::kBufs != Plain::kBufs;
        const int grid = groups * a.splits;
        if (WIDE && a.wide && a.vec) attend_few_kernel<T, DP, WIDE, true><<<grid, Wide::kWaves * 64, 0, s>>>(a, rows, G);
        else if (a.vec) attend_few_kernel<T, DP, false, true><<<grid, threads, 0, s>>>(a, rows, G);
        else attend_few_kernel<T, DP, false, false><<<grid, threads, 0, s>>>(a, rows, G);
    } else {
        const int tiles = (rows + 127) / 128, grid = groups * a.splits * tiles;
        if (a.vec) attend_rows_kernel<T, DP, BN, true><<<grid, kHeadsThreads, 0, s>>>(a, rows, G, tiles);
        else attend_rows_kernel<T, DP, BN, false><<<grid, kHeadsThreads, 0, s>>>(a, rows, G, tiles);
    }
}

template <typename T>
void attend_dim(const AttendArgs &a, int rows, int G, int groups, hipStream_t s) {
    switch (heads_pad(a.Dk, a.Dv)) {
        case 64:  attend<T, 64>(a, rows, G, groups, s); break;
        case 128: attend<T, 128>(a, rows, G, groups, s); break;
        default:  attend<T, 256>(a, rows, G, groups, s); break;
    }
}

}  // namespace
}  // namespace heads

hipError_t launch_attend(const AttendArgs &a, int dtype, hipStream_t s) {
    const int G = a.Hq / a.Hkv, rows = (a.shared ? a.B : 1) * a.Tq * G, groups = (a.shared ? 1 : a.B) * a.Hkv;
    if (dtype == SDPA_BF16) heads::attend_dim<__bf16>(a, rows, G, groups, s);
    else heads::attend_dim<float>(a, rows, G, groups, s);
    return hipGetLastError();
}

namespace heads {
namespace {
template <typename T> void combine(const AttendArgs &a, int slots, hipStream_t s) {
    const long rows = (long)a.B * a.Tq * a.Hq;
    const int groups = combine_groups(rows, slots);
    const unsigned grid = combine_blocks(rows, groups);
    if (groups == 8) combine_kernel<T, 8><<<grid, kHeadsThreads, 0, s>>>(a, slots);
    else combine_kernel<T, 1><<<grid, kHeadsThreads, 0, s>>>(a, slots);
}
template <typename T> void combine_scored(const AttendArgs &a, const WeightArgs &w, int slots, hipStream_t s) {
    const long rows = slots > 1 ? (long)a.B * a.Tq * a.Hq : 0;
    const int groups = combine_groups(rows, slots);
    const unsigned blocks = combine_blocks(rows, groups), grid = blocks + (unsigned)(a.B * a.Hkv * ((a.Tk + 1023) / 1024));
    if (groups == 8) combine_scored_kernel<T, 8><<<grid, kHeadsThreads, 0, s>>>(a, w, slots, (int)blocks);
    else combine_scored_kernel<T, 1><<<grid, kHeadsThreads, 0, s>>>(a, w, slots, (int)blocks);
}
}  // namespace
}  // namespace heads

hipError_t launch_combine(const AttendArgs &a, int slots, int dtype, hipStream_t s) {
    if (dtype == SDPA_BF16) heads::combine<__bf16>(a, slots, s);
    else heads::combine<float>(a, slots, s);
    return hipGetLastError();
}

hipError_t launch_combine_scored(const AttendArgs &a, const WeightArgs &w, int slots, int dtype, hipStream_t s) {
    if (dtype == SDPA_BF16) heads::combine_scored<__bf16>(a, w, slots, s);
    else heads::combine_scored<float>(a, w, slots, s);
    return hipGetLastError();
}

}  // namespace sdpa
