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
template <typename T, int DP>
__global__ __launch_bounds__(kHeadsThreads) void backward_rows_kernel(BackwardArgs a, int rows, int G, int tiles) {
    using TL = Tile<T, DP>;
    constexpr int BN = 32, STEPS = DP / Ops<T>::kStep;
    __shared__ __attribute__((aligned(1024))) char lk[BN * TL::kRowBytes];
    __shared__ __attribute__((aligned(1024))) char lv[BN * TL::kRowBytes];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
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
    const unsigned tk = lds_address(lk), ak = tk + map.rows, av = lds_address(lv) + map.rows;
    constexpr int PIECES = BN * TL::kChunks / kHeadsThreads;
    u32x4 rk[PIECES], rv[PIECES];
    const TileList list = tile_list(wg, a.sinks, BN);
    auto fetch = [&](int it) {
        const int j0 = list.at(it) * BN;
#pragma unroll
        for (int k = 0; k < PIECES; ++k) {
            const int c = tid + k * kHeadsThreads, j = j0 + c / TL::kChunks, d = (c % TL::kChunks) * Ops<T>::kVec;
            rk[k] = rv[k] = u32x4{0, 0, 0, 0};
            if (j < wg.hi_max && (j >= wg.lo_min || j < a.sinks)) {
                rk[k] = load_chunk((const T *)row_at(a.k, b, j, h, sizeof(T)), d, a.Dk, a.vec);
                rv[k] = load_chunk((const T *)row_at(a.v, b, j, h, sizeof(T)), d, a.Dv, a.vec);
            }
        }
    };
    if (list.count > 0) fetch(0);
    for (int it = 0; it < list.count; ++it) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < PIECES; ++k) {
            const int c = tid + k * kHeadsThreads, p = TL::chunk(c / TL::kChunks, c % TL::kChunks);
            *reinterpret_cast<u32x4 *>(lk + p) = rk[k];
            *reinterpret_cast<u32x4 *>(lv + p) = rv[k];
        }
        __syncthreads();
        const int j0 = list.at(it) * BN, j1 = j0 + BN;
        if (it + 1 < list.count) fetch(it + 1);
        if (j0 >= wv.hi_max || (j1 <= wv.lo_min && j0 >= a.sinks)) continue;
        const bool full = j1 <= wv.hi_min && (j0 >= wv.lo_max || j1 <= a.sinks);
        f32x16 s = {}, dp = {};
#pragma unroll
        for (int i = 0; i < STEPS; ++i) s = Ops<T>::mma(read_rows<T, DP>(ak, 0, i), q[i], s);
#pragma unroll
        for (int i = 0; i < STEPS; ++i) dp = Ops<T>::mma(read_rows<T, DP>(av, 0, i), g[i], dp);
        uint32_t vis = 0xffffu;
        if (!full) {
            vis = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int j = j0 + row_of(i, lane >> 5);
                if (j < seen.hi && (j >= seen.lo || j < a.sinks)) vis |= 1u << i;
            }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float p = __builtin_amdgcn_exp2f(s[i] * a.scale_log2 - lse2);
            s[i] = (vis >> i) & 1 ? p * (dp[i] - delta) : 0.f;
        }
        mma_block<T, DP, DP / 32>(dq, tk, map, 0, to_probs(s, T()), !full, vis, 1, lane);
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

// which rows (tokens' grouped heads) a key is seen by: [lo, hi)
struct SeenBy { int lo, hi; };
__device__ inline SeenBy seen_by(int j, int nq, int nk, int G, int window, int sinks) {
    SeenBy s = {0, 0};
    if (j >= nk || nq <= 0) return s;
    const int p0 = nk - nq;                             // the first query's position (below 0: it has seen nothing yet)
    const int lo = j - p0 > 0 ? j - p0 : 0;
    int hi = j < sinks || j - p0 + window > nq ? nq : j - p0 + window;
    if (hi < lo || lo > nq) hi = 0;
    if (hi == 0) return s;
    s.lo = lo * G; s.hi = hi * G;
    return s;
}

// ---- dK, dV: 128 keys to a workgroup, 32 to a wave ------------------------------------------------------------------------
// WHAT: 3 = both; fp32 rows of 256 do them one after the other (1 = dV, 2 = dK): two accumulators and two operands of 256
// columns do not fit the 512 registers of a lane.
template <typename T, int DP, int WHAT>
__global__ __launch_bounds__(kHeadsThreads) void backward_keys_kernel(BackwardArgs a, int rows, int G, int items) {
    using TL = Tile<T, DP>;
    constexpr int BQ = 32, STEPS = DP / Ops<T>::kStep;
    constexpr bool DV = (WHAT & 1) != 0, DK = (WHAT & 2) != 0;
    __shared__ __attribute__((aligned(1024))) char lq[BQ * TL::kRowBytes];
    __shared__ __attribute__((aligned(1024))) char lg[BQ * TL::kRowBytes];
    __shared__ float llse[BQ], ldelta[BQ];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int id = xcd_place(blockIdx.x, gridDim.x);
    const int item = id % items;
    id /= items;
    const int h = id % a.Hkv, b = id / a.Hkv;
    const int sink_items = a.sink_blocks * a.sink_chunks;
    const int chunks = item < sink_items ? a.sink_chunks : a.rest_chunks;
    const int block = item < sink_items ? item / chunks : a.sink_blocks + (item - sink_items) / chunks;
    const int chunk = item < sink_items ? item % chunks : (item - sink_items) % chunks;
    const int nq = clamp_len(a.q_lens, b, a.Tq), nk = clamp_len(a.kv_lens, b, a.Tk);
    const int k0 = block * kBwdKeys, kw = k0 + wave * 32, j = kw + (lane & 31);
    const SeenBy by = seen_by(j, nq, nk, G, a.window, a.sinks);
    // the rows that any of the workgroup's keys is seen by: contiguous, from the first key's first to the last key's last (or to
    // the end, with a sink key among them)
    const int klast = min(k0 + kBwdKeys, nk) - 1;
    SeenBy all = {0, 0};
    if (k0 < nk) {
        all = seen_by(k0, nq, nk, G, a.window, a.sinks);
        const SeenBy last = seen_by(klast, nq, nk, G, a.window, a.sinks);
        if (all.hi == 0) all.lo = max(0, k0 - (nk - nq)) * G;      // (the first keys may lie before every window)
        all.hi = max(all.hi, last.hi);
        if (k0 < a.sinks) all.hi = max(all.hi, seen_by(min(a.sinks - 1, klast), nq, nk, G, a.window, a.sinks).hi);
    }
    const int w_last = min(kw + 31, nk - 1);
    // rows that see every key of the wave: from the last key's first to the smallest end, which is the first key's that is no sink
    const int f_first_key = kw < a.sinks ? min(a.sinks, w_last) : kw;
    const SeenBy f_first = seen_by(f_first_key, nq, nk, G, a.window, a.sinks), f_last = seen_by(w_last, nq, nk, G, a.window, a.sinks);
    const int full_lo = f_last.lo, full_hi = kw + 32 <= nk ? min(f_first.hi, f_last.hi) : 0;
    const int n_tiles = all.hi > all.lo ? (all.hi - all.lo / BQ * BQ + BQ - 1) / BQ : 0;
    const int first = all.lo / BQ;
    const int it0 = (int)((long)n_tiles * chunk / chunks), it1 = (int)((long)n_tiles * (chunk + 1) / chunks);

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
    const unsigned tq = lds_address(lq), tg = lds_address(lg), aq = tq + map.rows, ag = tg + map.rows;
    constexpr int PIECES = BQ * TL::kChunks / kHeadsThreads;
    u32x4 rq[PIECES], rg[PIECES];
    float rl = 0.f, rd = 0.f;
    auto fetch = [&](int it) {
        const int r0 = (first + it) * BQ;
#pragma unroll
        for (int k = 0; k < PIECES; ++k) {
            const int c = tid + k * kHeadsThreads, r = r0 + c / TL::kChunks, d = (c % TL::kChunks) * Ops<T>::kVec;
            rq[k] = rg[k] = u32x4{0, 0, 0, 0};
            if (r < all.hi) {
                const int t = r / G, hq = h * G + r - t * G;
                rq[k] = load_chunk((const T *)row_at(a.q, b, t, hq, sizeof(T)), d, a.Dk, a.vec);
                rg[k] = load_chunk((const T *)row_at(a.dout, b, t, hq, sizeof(T)), d, a.Dv, a.vec);
            }
        }
        if (tid < BQ && r0 + tid < all.hi) {
            const int r = r0 + tid, t = r / G, hq = h * G + r - t * G;
            const long at = ((long)b * a.Hq + hq) * a.Tq + t;
            rl = a.lse[at] * kLog2e;
            rd = a.delta[at];
        }
    };
    if (it0 < it1) fetch(it0);
    for (int it = it0; it < it1; ++it) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < PIECES; ++k) {
            const int c = tid + k * kHeadsThreads, p = TL::chunk(c / TL::kChunks, c % TL::kChunks);
            *reinterpret_cast<u32x4 *>(lq + p) = rq[k];
            *reinterpret_cast<u32x4 *>(lg + p) = rg[k];
        }
        if (tid < BQ) { llse[tid] = rl; ldelta[tid] = rd; }
        __syncthreads();
        const int r0 = (first + it) * BQ;
        if (it + 1 < it1) fetch(it + 1);
        const bool full = r0 >= full_lo && r0 + BQ <= full_hi;
        f32x16 s = {};
#pragma unroll
        for (int i = 0; i < STEPS; ++i) s = Ops<T>::mma(read_rows<T, DP>(aq, 0, i), kf[i], s);
        uint32_t vis = 0xffffu;
        if (!full) {
            vis = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int r = r0 + row_of(i, lane >> 5);
                if (r >= by.lo && r < by.hi) vis |= 1u << i;
            }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float p = __builtin_amdgcn_exp2f(s[i] * a.scale_log2 - llse[row_of(i, lane >> 5)]);
            s[i] = (vis >> i) & 1 ? p : 0.f;
        }
        if constexpr (DV) mma_block<T, DP, DP / 32>(dv, tg, map, 0, to_probs(s, T()), !full, vis, 1, lane);
        if constexpr (DK) {
            f32x16 dp = {};
#pragma unroll
            for (int i = 0; i < STEPS; ++i) dp = Ops<T>::mma(read_rows<T, DP>(ag, 0, i), vf[i], dp);
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = (vis >> i) & 1 ? s[i] * (dp[i] - ldelta[row_of(i, lane >> 5)]) : 0.f;
            mma_block<T, DP, DP / 32>(dk, tq, map, 0, to_probs(s, T()), !full, vis, 1, lane);
        }
    }
    if (j >= a.Tk) return;
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

// the chunks of a key block become its gradient: a workgroup per key block, the chunks added in their order
template <typename T>
__global__ __launch_bounds__(kHeadsThreads) void backward_join_kernel(BackwardArgs a, int block0, int blocks, long item0, int chunks,
                                                                      long per) {
    int id = blockIdx.x;
    const int blk = id % blocks;
    id /= blocks;
    const int h = id % a.Hkv, b = id / a.Hkv, k0 = (block0 + blk) * kBwdKeys, w = a.Dk + a.Dv;
    const float *src = a.part + (((long)b * a.Hkv + h) * per + item0 + (long)blk * chunks) * kBwdKeys * w;
    for (int i = threadIdx.x; i < kBwdKeys * w; i += kHeadsThreads) {
        const int key = i / w, c = i - key * w, j = k0 + key;
        if (j >= a.Tk) break;
        float sum = 0.f;
        for (int x = 0; x < chunks; ++x) sum += src[(long)x * kBwdKeys * w + i];
        T *row = c < a.Dk ? (T *)row_at(a.dk, b, j, h, sizeof(T)) + c : (T *)row_at(a.dv, b, j, h, sizeof(T)) + (c - a.Dk);
        *row = from_f32<T>(sum);
    }
}

// ---- the weights of every key: 128 keys to a workgroup ------------------------------------------------------------------------
// w_out_j = w_in_j + sum_i exp(s_ij - lse_i): the first half of the dK / dV walk, with column sums in place of the products.
template <typename T, int DP>
__global__ __launch_bounds__(kHeadsThreads) void weights_kernel(WeightArgs a, int G, int blocks) {
    using TL = Tile<T, DP>;
    constexpr int BQ = 32, STEPS = DP / Ops<T>::kStep;
    __shared__ __attribute__((aligned(1024))) char lq[BQ * TL::kRowBytes];
    __shared__ float llse[BQ];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int id = xcd_place(blockIdx.x, gridDim.x);
    const int k0 = (id % blocks) * kBwdKeys, kw = k0 + wave * 32, j = kw + (lane & 31);
    id /= blocks;
    const int h = id % a.Hkv, b = id / a.Hkv;
    const int nq = clamp_len(a.q_lens, b, a.Tq), nk = clamp_len(a.kv_lens, b, a.Tk);
    const int everything = 1 << 30;
    const SeenBy by = seen_by(j, nq, nk, G, everything, 0);
    float sum = 0.f;
    if (k0 < nk) {
        const SeenBy first = seen_by(k0, nq, nk, G, everything, 0);
        const int r_end = nq * G;
        typename Ops<T>::Frag kf[STEPS];
        load_row<T, DP>(kf, row_at(a.k, b, j, h, sizeof(T)), a.Dk, j < nk, a.vec, lane);
        LaneMap<T, DP> map;
        map.init(lane);
        const unsigned aq = lds_address(lq) + map.rows;
        for (int r0 = first.lo / BQ * BQ; r0 < r_end; r0 += BQ) {
            __syncthreads();
            for (int c = tid; c < BQ * TL::kChunks; c += kHeadsThreads) {
                const int r = r0 + c / TL::kChunks;
                u32x4 x = {0, 0, 0, 0};
                if (r < r_end) {
                    const int t = r / G, hq = h * G + r - t * G;
                    x = load_chunk((const T *)row_at(a.q, b, t, hq, sizeof(T)), (c % TL::kChunks) * Ops<T>::kVec, a.Dk, a.vec);
                }
                *reinterpret_cast<u32x4 *>(lq + TL::chunk(c / TL::kChunks, c % TL::kChunks)) = x;
            }
            if (tid < BQ && r0 + tid < r_end) {
                const int r = r0 + tid, t = r / G, hq = h * G + r - t * G;
                llse[tid] = a.lse[((long)b * a.Hq + hq) * a.Tq + t] * kLog2e;
            }
            __syncthreads();
            f32x16 s = {};
#pragma unroll
            for (int i = 0; i < STEPS; ++i) s = Ops<T>::mma(read_rows<T, DP>(aq, 0, i), kf[i], s);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int rl = row_of(i, lane >> 5), r = r0 + rl;
                if (r >= by.lo && r < by.hi) sum += __builtin_amdgcn_exp2f(s[i] * a.scale_log2 - llse[rl]);
            }
        }
    }
    sum = half_sum(sum);
    if (lane < 32 && j < a.Tk) {
        const float w = a.w_in[b * a.wi_batch + h * a.wi_head + j];
        a.w_out[b * a.wo_batch + h * a.wo_head + j] = w + sum;
    }
}

template <typename T, int DP>
void backward(const BackwardArgs &a, hipStream_t s) {
    const int G = a.Hq / a.Hkv, rows = a.Tq * G, groups = a.B * a.Hkv;
    const int tiles = (rows + kBwdRows - 1) / kBwdRows;
    if (tiles > 0) backward_rows_kernel<T, DP><<<groups * tiles, kHeadsThreads, 0, s>>>(a, rows, G, tiles);
    const int blocks = (a.Tk + kBwdKeys - 1) / kBwdKeys, rest = blocks - a.sink_blocks;
    const int sink_items = a.sink_blocks * a.sink_chunks, items = sink_items + rest * a.rest_chunks;
    if (items == 0) return;
    if constexpr (DP * (int)sizeof(T) > 512) {
        backward_keys_kernel<T, DP, 1><<<groups * items, kHeadsThreads, 0, s>>>(a, rows, G, items);
        backward_keys_kernel<T, DP, 2><<<groups * items, kHeadsThreads, 0, s>>>(a, rows, G, items);
    } else {
        backward_keys_kernel<T, DP, 3><<<groups * items, kHeadsThreads, 0, s>>>(a, rows, G, items);
    }
    const long base = a.sink_chunks > 1 ? 0 : sink_items, per = items - base - (a.rest_chunks > 1 ? 0 : items - sink_items);
    if (a.sink_chunks > 1 && a.sink_blocks > 0)
        backward_join_kernel<T><<<groups * a.sink_blocks, kHeadsThreads, 0, s>>>(a, 0, a.sink_blocks, 0, a.sink_chunks, per);
    if (a.rest_chunks > 1 && rest > 0)
        backward_join_kernel<T><<<groups * rest, kHeadsThreads, 0, s>>>(a, a.sink_blocks, rest, sink_items - base, a.rest_chunks, per);
}

template <typename T, int DP>
void weights(const WeightArgs &a, hipStream_t s) {
    const int blocks = (a.Tk + kBwdKeys - 1) / kBwdKeys;
    if (blocks > 0) weights_kernel<T, DP><<<a.B * a.Hkv * blocks, kHeadsThreads, 0, s>>>(a, a.Hq / a.Hkv, blocks);
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
