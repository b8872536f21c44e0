// sdpa_heads_device.h -- device pieces the batched attention kernels share.
//
// Every product here is D = A * B with a 32x32 MFMA, whose result a lane holds as one COLUMN (lane & 31) and the 16 rows
// (i & 3) + 8 * (i >> 2) + 4 * (lane >> 5).  Two products in a row keep their middle operand in registers: the
// probabilities of one column, read as the B operand of the next product, need the inner index in exactly the order the
// rows already have -- inner slot (half h, element e) is row 8 * (e >> 2) + 4 * h + (e & 3) of a 16-row group -- and the other
// operand is read from LDS in that same order (the inner index of a product may be permuted freely, as long as both
// operands agree).  For bf16 that read is the transposing LDS load, which hands a lane four rows of its column.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "sdpa_heads.h"

namespace sdpa {
namespace heads {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kHeadsThreads = 256;
constexpr float kLn2 = 0.693147180559945309f, kLog2e = 1.44269504088896341f;
constexpr float kNegInf = -__builtin_inff();

using LdsVec4 = __attribute__((address_space(3))) s16x4;

__device__ inline int row_of(int i, int half) { return (i & 3) + 8 * (i >> 2) + 4 * half; }

template <typename T> struct Ops;

template <> struct Ops<__bf16> {
    using Frag = bf16x8;
    static constexpr int kVec = 8;                 // elements of a 16-byte chunk
    static constexpr int kStep = 16;               // inner elements one step (both lane halves) covers
    __device__ static f32x16 mma(Frag a, Frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};

template <> struct Ops<float> {
    using Frag = f32x4;
    static constexpr int kVec = 4;
    static constexpr int kStep = 8;
    __device__ static f32x16 mma(Frag a, Frag b, f32x16 c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
};

__device__ inline float to_f32(__bf16 x) { return (float)x; }
__device__ inline float to_f32(float x) { return x; }
template <typename T> __device__ inline T from_f32(float x) { return (T)x; }   // (to nearest even)

// ---- LDS tiles: rows of DP elements, 16-byte chunks XOR-swizzled by the row ----------------------------------------------
// Both readers are conflict-free: 16 consecutive rows at one chunk (the row-wise fragments) land in 16 different chunk
// classes of the 64 banks, and 4 consecutive rows at 4 consecutive chunks (the transposing load) do too.
template <typename T, int DP> struct Tile {
    static constexpr int kChunks = DP * (int)sizeof(T) / 16;
    static constexpr int kRowBytes = DP * (int)sizeof(T);
    __device__ static int swz(int row) {
        return kChunks == 8 ? (((row >> 1) & 1) << 2) | ((row >> 2) & 3) : ((row & 3) << 2) | ((row >> 2) & 3);
    }
    __device__ static int chunk(int row, int c) { return row * kRowBytes + ((c ^ swz(row)) << 4); }
    __device__ static int elem(int row, int col) {
        const int b = col * (int)sizeof(T);
        return chunk(row, b >> 4) + (b & 15);
    }
};

// 16 bytes of a row: elements [d0, d0 + kVec), zero from `dim` on
template <typename T> __device__ inline u32x4 load_chunk(const T *row, int d0, int dim, bool vec) {
    constexpr int N = Ops<T>::kVec;
    u32x4 r = {0, 0, 0, 0};
    if (vec) {
        if (d0 < dim) r = *reinterpret_cast<const u32x4 *>(row + d0);
    } else {
        union { T e[N]; u32x4 u; } x;
        x.u = r;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (d0 + i < dim) x.e[i] = row[d0 + i];
        r = x.u;
    }
    return r;
}

// A fragment (a lane's 16 bytes of step s of row lane & 31) of a tile's 32-row block
template <typename T, int DP> __device__ inline typename Ops<T>::Frag read_rows(const char *tile, int block, int s, int lane) {
    return *reinterpret_cast<const typename Ops<T>::Frag *>(tile + Tile<T, DP>::chunk(block * 32 + (lane & 31), 2 * s + (lane >> 5)));
}

// The transposed operand of a 32-row block: columns col0 .. col0 + 31, all 32 rows as the inner index.
template <typename T> struct Cols;                 // 32 rows of one column in product order
template <> struct Cols<__bf16> { bf16x8 f[2]; };
template <> struct Cols<float> { float f[16]; };

template <int DP> __device__ inline Cols<__bf16> read_cols(const char *tile, int block, int col0, int lane, __bf16) {
    Cols<__bf16> r;
    const int col = col0 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3), half = lane >> 5, sub = (lane & 15) >> 2;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
        union { s16x4 h[2]; bf16x8 f; } x;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int row = block * 32 + 16 * ks + 8 * e + 4 * half + sub;
            x.h[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsVec4 *)(tile + Tile<__bf16, DP>::elem(row, col)));
        }
        r.f[ks] = x.f;
    }
    return r;
}
template <int DP> __device__ inline Cols<float> read_cols(const char *tile, int block, int col0, int lane, float) {
    Cols<float> r;
#pragma unroll
    for (int i = 0; i < 16; ++i)
        r.f[i] = *reinterpret_cast<const float *>(tile + Tile<float, DP>::elem(block * 32 + row_of(i, lane >> 5), col0 + (lane & 31)));
    return r;
}

// 16 values of a lane's column as the B operand of the next product
template <typename T> struct Probs;
template <> struct Probs<__bf16> { bf16x8 f[2]; };
template <> struct Probs<float> { float f[16]; };
// Rounded to bf16: the operand type of the matrix instructions.  A weight is off by at most 2^-8 of itself, independently
// of its neighbours; the sums that normalise them are taken before the rounding, in 32 bits.
__device__ inline Probs<__bf16> to_probs(const f32x16 &p, __bf16) {
    Probs<__bf16> r;
#pragma unroll
    for (int i = 0; i < 16; ++i) r.f[i >> 3][i & 7] = (__bf16)p[i];
    return r;
}
__device__ inline Probs<float> to_probs(const f32x16 &p, float) {
    Probs<float> r;
#pragma unroll
    for (int i = 0; i < 16; ++i) r.f[i] = p[i];
    return r;
}

__device__ inline f32x16 mma_cols(const Cols<__bf16> &a, const Probs<__bf16> &b, f32x16 c) {
    c = Ops<__bf16>::mma(a.f[0], b.f[0], c);
    return Ops<__bf16>::mma(a.f[1], b.f[1], c);
}
__device__ inline f32x16 mma_cols(const Cols<float> &a, const Probs<float> &b, f32x16 c) {
#pragma unroll
    for (int i = 0; i < 16; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.f[i], b.f[i], c, 0, 0, 0);
    return c;
}

// ---- values that are no numbers behind a mask ---------------------------------------------------------------------------
// A masked pair has weight 0, and 0 * NaN would still be NaN in the product's sum.  Where a block holds masked pairs its
// operand is looked at first: values that are not finite leave the product (as zeros) and come back only for the columns that
// see them, by a second product of 0/1 indicators.  `kinds`: 3 = NaN, +inf and -inf apart (weights are positive, so the sum's
// sign is theirs), 1 = all of them as NaN (gradients, whose weights have either sign).
template <typename T, int DP> __device__ inline bool block_not_finite(const char *tile, int block, int lane) {
    const u32x4 *at = reinterpret_cast<const u32x4 *>(tile + block * 32 * Tile<T, DP>::kRowBytes) + lane;
    uint32_t bad = 0;
#pragma unroll 4
    for (int k = 0; k < 32 * Tile<T, DP>::kChunks / 64; ++k) {
        const u32x4 w = at[k * 64];
#pragma unroll
        for (int i = 0; i < 4; ++i)      // an exponent of all ones carries into the sign's place
            bad |= sizeof(T) == 2 ? ((w[i] & 0x7f807f80u) + 0x00800080u) & 0x80008000u : ((w[i] & 0x7f800000u) + 0x00800000u) & 0x80000000u;
    }
    return __any(bad != 0);
}
// kind 0: the finite values; 1: NaN (kinds == 1: anything not finite); 2: +inf; 3: -inf -- 1.0 there, 0 elsewhere
__device__ inline float pick(float x, int kind, int kinds) {
    const uint32_t u = __float_as_uint(x);
    const bool fin = (u & 0x7f800000u) != 0x7f800000u;
    if (kind == 0) return fin ? x : 0.f;
    if (kind == 1) return (kinds == 1 ? !fin : (u & 0x7fffffffu) > 0x7f800000u) ? 1.f : 0.f;
    return u == (kind == 2 ? 0x7f800000u : 0xff800000u) ? 1.f : 0.f;
}
__device__ inline Cols<__bf16> pick(const Cols<__bf16> &a, int kind, int kinds) {
    Cols<__bf16> r;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int i = 0; i < 8; ++i) r.f[ks][i] = (__bf16)pick((float)a.f[ks][i], kind, kinds);
    return r;
}
__device__ inline Cols<float> pick(const Cols<float> &a, int kind, int kinds) {
    Cols<float> r;
#pragma unroll
    for (int i = 0; i < 16; ++i) r.f[i] = pick(a.f[i], kind, kinds);
    return r;
}

// acc += A * P where A holds values that are not finite; `seen` = bit i set where the lane's column sees row i
template <typename T>
__device__ inline f32x16 mma_cols_guarded(const Cols<T> &a, const Probs<T> &b, uint32_t seen, int kinds, f32x16 c) {
    f32x16 one;
#pragma unroll
    for (int i = 0; i < 16; ++i) one[i] = (seen >> i) & 1 ? 1.f : 0.f;
    const Probs<T> vis = to_probs(one, T());
    c = mma_cols(pick(a, 0, kinds), b, c);
#pragma unroll 1
    for (int kind = 1; kind <= kinds; ++kind) {
        f32x16 n = {};
        n = mma_cols(pick(a, kind, kinds), vis, n);
        const float add = kind == 1 ? __builtin_nanf("") : kind == 2 ? __builtin_inff() : kNegInf;
#pragma unroll
        for (int i = 0; i < 16; ++i) c[i] += n[i] > 0.f ? add : 0.f;
    }
    return c;
}

// acc[d] += (columns d * 32 .. of the block)^T * P for every d < N; masked: the block holds masked pairs
template <typename T, int DP, int N>
__device__ inline void mma_block(f32x16 *acc, const char *tile, int block, const Probs<T> &p, bool masked, uint32_t seen,
                                 int kinds, int lane) {
    if (masked && block_not_finite<T, DP>(tile, block, lane)) {
        // (a rare path: one body for every d, the accumulators handed round, so that it costs the other path no registers)
#pragma unroll 1
        for (int d = 0; d < N; ++d) {
            const f32x16 t = mma_cols_guarded<T>(read_cols<DP>(tile, block, d * 32, lane, T()), p, seen, kinds, acc[0]);
#pragma unroll
            for (int e = 0; e + 1 < N; ++e) acc[e] = acc[e + 1];
            acc[N - 1] = t;
        }
    } else {
#pragma unroll
        for (int d = 0; d < N; ++d) acc[d] = mma_cols(read_cols<DP>(tile, block, d * 32, lane, T()), p, acc[d]);
    }
}

// ---- which keys a query sees ------------------------------------------------------------------------------------------
// Key j is visible to a row when j < hi and (j >= lo or j < sinks); hi = 0 for a row that does not exist.
struct Seen { int hi, lo; };
// the same for a run of rows: smallest and largest of either bound over the rows that exist (hi_max = 0: none does)
struct SeenRange { int hi_min, hi_max, lo_min, lo_max; };

__device__ inline int clamp_len(const int *lens, int b, int cap) {
    if (!lens) return cap;
    const int n = lens[b];
    return n < 0 ? 0 : n > cap ? cap : n;
}
__device__ inline Seen seen_at(int pos, int nk, int window) {
    Seen s;
    s.hi = pos + 1 < nk ? pos + 1 : nk;
    if (s.hi < 0) s.hi = 0;
    s.lo = pos - window + 1;
    if (s.lo < 0) s.lo = 0;
    return s;
}
// tokens t0 .. t1 (inclusive) of a sequence with nq queries and nk keys
__device__ inline SeenRange seen_range(int t0, int t1, int nq, int nk, int window) {
    SeenRange r = {0, 0, 0, 0};
    if (t1 > nq - 1) t1 = nq - 1;
    if (t1 < t0) return r;
    const Seen a = seen_at(nk - nq + t0, nk, window), b = seen_at(nk - nq + t1, nk, window);
    r.hi_min = a.hi; r.hi_max = b.hi; r.lo_min = a.lo; r.lo_max = b.lo;
    return r;
}
// the key tiles a run of rows visits: [0, sink_tiles) and [first, end) -- ONE list of `count`, never a tile twice
struct TileList {
    int sink_tiles, first, count;
    __device__ int at(int i) const { return i < sink_tiles ? i : first + (i - sink_tiles); }
};
__device__ inline TileList tile_list(const SeenRange &r, int sinks, int bn) {
    TileList l;
    const int sh = sinks < r.hi_max ? sinks : r.hi_max;
    l.sink_tiles = (sh + bn - 1) / bn;
    l.first = r.lo_min / bn;
    if (l.first < l.sink_tiles) l.first = l.sink_tiles;
    const int end = r.lo_min < r.hi_max ? (r.hi_max + bn - 1) / bn : 0;
    l.count = l.sink_tiles + (end > l.first ? end - l.first : 0);
    return l;
}

// Consecutive workgroups go to the 8 XCDs in turn, and each XCD has an L2 of its own: workgroups that read the same keys are
// given consecutive places on ONE of them.
__device__ inline int xcd_place(int id, int n) {
    const int per = n >> 3;
    return id < per * 8 ? (id & 7) * per + (id >> 3) : id;
}

__device__ inline float half_max(float x) { return fmaxf(x, __shfl_xor(x, 32)); }
__device__ inline float half_sum(float x) { return x + __shfl_xor(x, 32); }

}  // namespace heads
}  // namespace sdpa
