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
#include "sdpa_internal.h"

namespace sdpa {
namespace heads {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kHeadsThreads = 256;
constexpr float kLn2 = 0.693147180559945309f, kLog2e = 1.44269504088896341f;
constexpr float kNegInf = -__builtin_inff();

using LdsVec4 = __attribute__((address_space(3))) s16x4;

// A copy the compiler knows nothing about: what is computed from it stays where it is used.  In the kernels' rarer branches, whose lane
// arithmetic would otherwise be moved in front of the loops and hold the registers that the frequent branch needs.
__device__ inline int opaque(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

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
// Chunk c of a row lies at row * kRowBytes + ((c ^ swz(row)) << 4): LaneMap reads by this, the stagers write by it.
// Both readers are conflict-free: 16 consecutive rows at one chunk (the row-wise fragments) land in 16 different chunk
// classes of the 64 banks, and 4 consecutive rows at 4 consecutive chunks (the transposing load) do too.
template <typename T, int DP> struct Tile {
    static constexpr int kChunks = DP * (int)sizeof(T) / 16;
    static constexpr int kRowBytes = DP * (int)sizeof(T);
    __device__ static int swz(int row) {
        return kChunks == 8 ? (((row >> 1) & 1) << 2) | ((row >> 2) & 3) : ((row & 3) << 2) | ((row >> 2) & 3);
    }
};

// 16 bytes of a row: elements [d0, d0 + kVec), zero from `dim` on.  `vec`: the row is 16-byte aligned and whole.  Others, in
// bf16, are read in one load too (at their elements' alignment, which global loads allow), but for the row's last piece, whose elements are
// read at once: two sequences of 1024 tokens, 8 heads of 100 columns, window 300, backward 169 us (element by element throughout: 284).  For
// fp32's four elements that gains 5 % and costs the widest heads registers.
template <typename T> __device__ inline u32x4 load_chunk(const T *row, int d0, int dim, bool vec) {
    constexpr int N = Ops<T>::kVec;
    u32x4 r = {0, 0, 0, 0};
    if (vec) {
        if (d0 < dim) r = *reinterpret_cast<const u32x4 *>(row + d0);
    } else if (sizeof(T) == 4) {
        union { T e[N]; u32x4 u; } x;
        x.u = r;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (d0 + i < dim) x.e[i] = row[d0 + i];
        r = x.u;
    } else if (d0 + N <= dim) {
        __builtin_memcpy(&r, row + d0, 16);
    } else if (d0 < dim) {
        union { T e[N]; u32x4 u; } x;
#pragma unroll
        for (int i = 0; i < N; ++i) x.e[i] = row[min(d0 + i, dim - 1)];
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (d0 + i >= dim) x.e[i] = T(0.f);
        r = x.u;
    }
    return r;
}

// Where a lane reads, as byte addresses inside a tile.  The swizzle is an XOR of the chunk number, so every read of a lane is ONE
// base address, XORed with a constant (the step or column block: bits 4..7) plus a constant (the block: an immediate of the
// instruction); tiles begin at multiples of 256 bytes.
template <typename T, int DP> struct LaneMap {
    using TL = Tile<T, DP>;
    unsigned rows;                       // row-wise: row lane & 31, the lane half's chunk
    unsigned cols;                       // transposed: rows 4 * half + sub (bf16) / 4 * half (fp32), the lane's columns
    __device__ void init(int lane) {
        const int half = lane >> 5, row = lane & 31;
        rows = (unsigned)(row * TL::kRowBytes + ((half ^ TL::swz(row)) << 4));
        if (sizeof(T) == 2) {
            const int sub = (lane & 15) >> 2, c = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), r = 4 * half + sub;
            cols = (unsigned)(r * TL::kRowBytes + ((c ^ TL::swz(r)) << 4) + (lane & 1) * 8);
        } else {
            cols = (unsigned)(4 * half * TL::kRowBytes + ((((lane & 31) >> 2) ^ TL::swz(4 * half)) << 4) + (lane & 3) * 4);
        }
    }
};
template <typename V> __device__ inline V lds_read(unsigned at, int offset) {
    return *(__attribute__((address_space(3))) const V *)((__attribute__((address_space(3))) const char *)(uintptr_t)at + offset);
}

// A fragment (a lane's 16 bytes of step s) of a tile's 32-row block; `at` = the tile's address + LaneMap::rows
template <typename T, int DP> __device__ inline typename Ops<T>::Frag read_rows(unsigned at, int block, int s) {
    using TL = Tile<T, DP>;
    constexpr int M = TL::kChunks < 16 ? TL::kChunks - 1 : 15;
    return lds_read<typename Ops<T>::Frag>(at ^ (unsigned)(((2 * s) & M) << 4), block * 32 * TL::kRowBytes + ((2 * s) & ~M) * 16);
}

// The transposed operand of a 32-row block: columns col0 .. col0 + 31, all 32 rows as the inner index.
template <typename T> struct Cols;                 // 32 rows of one column in product order
template <> struct Cols<__bf16> { bf16x8 f[2]; };
template <> struct Cols<float> { float f[16]; };

// `at` = the tile's address + LaneMap::cols; column block d = columns 32 d .. 32 d + 31.  In pieces of 16 bytes: bf16 the 16-row half
// `part`, fp32 the rows row_of(4 part .. 4 part + 3).
template <int DP> __device__ inline bf16x8 read_cols_part(unsigned at, int block, int d, int part, __bf16) {
    using TL = Tile<__bf16, DP>;
    union { s16x4 h[2]; bf16x8 f; } x;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const unsigned p = at ^ (unsigned)((((4 * d) & 15) ^ (2 * e)) << 4);      // (rows 8 e further: bit 1 of the swizzle)
        const int offset = (block * 32 + 16 * part + 8 * e) * TL::kRowBytes + ((4 * d) & ~15) * 16;
        x.h[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsVec4 *)((__attribute__((address_space(3))) char *)(uintptr_t)p + offset));
    }
    return x.f;
}
template <int DP> __device__ inline f32x4 read_cols_part(unsigned at, int block, int d, int part, float) {
    using TL = Tile<float, DP>;
    f32x4 f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = row_of(4 * part + i, 0), c = 8 * d;
        f[i] = lds_read<float>(at ^ (unsigned)(((c & 15) ^ TL::swz(row)) << 4), (block * 32 + row) * TL::kRowBytes + (c & ~15) * 16);
    }
    return f;
}
template <int DP> __device__ inline Cols<__bf16> read_cols(unsigned at, int block, int d, __bf16) {
    Cols<__bf16> r;
#pragma unroll
    for (int k = 0; k < 2; ++k) r.f[k] = read_cols_part<DP>(at, block, d, k, __bf16());
    return r;
}
template <int DP> __device__ inline Cols<float> read_cols(unsigned at, int block, int d, float) {
    Cols<float> r;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const f32x4 f = read_cols_part<DP>(at, block, d, k, float());
#pragma unroll
        for (int i = 0; i < 4; ++i) r.f[4 * k + i] = f[i];
    }
    return r;
}

// 16 values of a lane's column as the B operand of the next product.  bf16: in two terms, the value rounded and what that left of it, rounded
// (the operand type of the matrix instructions is bf16; half a step is 2^-8 of a value, so the two are off by 2^-16), and a product is two
// matrix instructions.  The sums that normalise them are taken before the rounding, in 32 bits.  With one term outputs are off by 0.0023
// of their norm and gradients by 0.0024, where the rounding of the results alone is 0.00166; with two it is 0.00166 and 0.00168.  What that
// costs (one term -> two): a prompt of 8192 tokens 194 -> 240 us, its gradients' training shape 337 -> 395, 64 tokens behind a prefix
// 74 -> 82; single tokens wait for the cache, 158 -> 160.
template <typename T> struct Probs;
template <> struct Probs<__bf16> { bf16x8 f[2], rest[2]; };
template <> struct Probs<float> { float f[16]; };
// value i (bf16: and i - 1) takes its place
__device__ inline void put_prob(Probs<__bf16> &p, const f32x16 &s, int i) {
#pragma clang fp contract(off)                           // (the value as it is summed, also where it comes from a product)
    const f32x2 v = {s[i - 1], s[i]};
    const bf16x2 x = __builtin_convertvector(v, bf16x2);
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const f32x2 left = {v[0] - __uint_as_float(u << 16), v[1] - __uint_as_float(u & 0xffff0000u)};
    const bf16x2 y = __builtin_convertvector(left, bf16x2);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        p.f[i >> 3][(i & 7) - 1 + k] = x[k];
        p.rest[i >> 3][(i & 7) - 1 + k] = y[k];
    }
}
__device__ inline void put_prob(Probs<float> &p, const f32x16 &s, int i) { p.f[i] = s[i]; }
__device__ inline Probs<__bf16> to_probs(const f32x16 &p, __bf16) {
    Probs<__bf16> r;
#pragma unroll
    for (int i = 1; i < 16; i += 2) put_prob(r, p, i);
    return r;
}
__device__ inline Probs<float> to_probs(const f32x16 &p, float) {
    Probs<float> r;
#pragma unroll
    for (int i = 0; i < 16; ++i) r.f[i] = p[i];
    return r;
}

__device__ inline f32x16 mma_part(bf16x8 a, const Probs<__bf16> &b, int part, f32x16 c) {
    c = Ops<__bf16>::mma(a, b.f[part], c);
    return Ops<__bf16>::mma(a, b.rest[part], c);
}
__device__ inline f32x16 mma_part(f32x4 a, const Probs<float> &b, int part, f32x16 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b.f[4 * part + i], c, 0, 0, 0);
    return c;
}
__device__ inline f32x16 mma_cols(const Cols<__bf16> &a, const Probs<__bf16> &b, f32x16 c) {
    c = mma_part(a.f[0], b, 0, c);
    return mma_part(a.f[1], b, 1, c);
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
template <typename T, int DP> __device__ inline bool block_not_finite(unsigned tile, int block, int lane) {
    const unsigned at = tile + (unsigned)(opaque(lane) * 16);
    // (0 * x is NaN for what is not finite, and 0 otherwise: one instruction for two bf16 values)
    float bad = 0.f;
#pragma unroll 4
    for (int k = 0; k < 32 * Tile<T, DP>::kChunks / 64; ++k) {
        const u32x4 w = lds_read<u32x4>(at + (unsigned)(k * 1024), block * 32 * Tile<T, DP>::kRowBytes);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t x = w[i];                     // (a variable of its own: a bit cast of a vector's element takes element 0)
            if constexpr (sizeof(T) == 2) bad = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, x), bf16x2{0, 0}, bad, false);
            else bad = __builtin_fmaf(__uint_as_float(x), 0.f, bad);
        }
    }
    return __any(bad != bad);
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

// acc[d] += (columns d * 32 .. of the block)^T * P for every d < N, where the block holds values that are not finite.
// (A rare path: one body for every d, the accumulators handed round, so that it costs the frequent path no registers.)
template <typename T, int DP, int N>
__device__ inline void mma_block_guarded(f32x16 *acc, unsigned tile, const LaneMap<T, DP> &map, int block, const Probs<T> &p,
                                         uint32_t seen, int kinds) {
#pragma unroll 1
    for (int d = 0; d < N; ++d) {
        // (the column block as a run-time number: its place is the XOR and the offset of read_cols at d = 0)
        const int c = d * 32 * (int)sizeof(T) / 16;
        const unsigned at = (tile + (unsigned)opaque((int)map.cols)) ^ (unsigned)((c & 15) << 4);
        const f32x16 t = mma_cols_guarded<T>(read_cols<DP>(at + (unsigned)((c & ~15) * 16), block, 0, T()), p, seen, kinds, acc[0]);
#pragma unroll
        for (int e = 0; e + 1 < N; ++e) acc[e] = acc[e + 1];
        acc[N - 1] = t;
    }
}

// the same, masked: the block holds masked pairs
template <typename T, int DP, int N>
__device__ inline void mma_block(f32x16 *acc, unsigned tile, const LaneMap<T, DP> &map, int block, const Probs<T> &p, bool masked,
                                 uint32_t seen, int kinds, int lane) {
    if (masked && __builtin_expect(block_not_finite<T, DP>(tile, block, lane), 0)) {
        mma_block_guarded<T, DP, N>(acc, tile, map, block, p, seen, kinds);
    } else {
        const unsigned at = tile + map.cols;
#pragma unroll
        for (int d = 0; d < N; ++d) acc[d] = mma_cols(read_cols<DP>(at, block, d, T()), p, acc[d]);
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
// The keys a run of rows visits as ONE list without a gap: the sinks, then the window from its first key on (or, where the two meet,
// everything from key 0) -- so that tiles begin at the window's first key and the sinks share a tile with it.
// A tile of the list is looked at in a frame: its row r is key j0 + r and sinks are what lies below `sinks` -- true for the tiles on
// either side, and for the tile with both (j0 counted back from the window) the sink rows lie below the window's first key.
struct Frame { int j0, sinks; };
struct KeyList {
    int s, shift, n;                 // entries below s are keys 0 .. s - 1, the others entry + shift; n entries
    int sinks;
    __device__ int tiles(int rows) const { return (n + rows - 1) / rows; }
    __device__ int key(int v) const { return v < s ? v : v + shift; }
    __device__ Frame frame(int v0, int rows) const {
        return s == 0 || v0 + rows <= s ? Frame{v0 + (s == 0 ? shift : 0), sinks} : Frame{v0 + shift, s + shift};
    }
};
__device__ inline KeyList key_list(const SeenRange &r, int sinks) {
    KeyList l;
    const int sh = sinks < r.hi_max ? sinks : r.hi_max, lo = r.lo_min < r.hi_max ? r.lo_min : r.hi_max;
    const bool gap = sh < lo;
    l.s = gap ? sh : 0;
    l.shift = gap ? lo - sh : 0;
    l.n = gap ? sh + r.hi_max - lo : r.hi_max;
    l.sinks = sinks;
    return l;
}
// does a run of rows see the frame's tile at all / all of it
__device__ inline bool sees_some(const SeenRange &w, Frame f, int rows) {
    return f.j0 < w.hi_max && (f.j0 + rows > w.lo_min || f.j0 < f.sinks);
}
__device__ inline bool sees_all(const SeenRange &w, Frame f, int rows) {
    return f.j0 + rows <= w.hi_min && (f.j0 >= w.lo_max || f.j0 + rows <= f.sinks);
}

// Consecutive workgroups go to the 8 XCDs in turn, and each XCD has an L2 of its own: workgroups that read the same keys are
// given consecutive places on ONE of them.
__device__ inline int xcd_place(int id, int n) {
    const int per = n >> 3;
    return id < per * 8 ? (id & 7) * per + (id >> 3) : id;
}

// a lane's value and the other half's at the same column
__device__ inline float half_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float half_sum(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// ---- key / value tiles from memory to LDS ---------------------------------------------------------------------------------
// One wave instruction moves 1 KiB (16 bytes a lane) straight to LDS, lane-linear at its LDS end; the tile's swizzle is made at
// the memory end, by the order in which the lanes ask for their row's chunks.  A lane's offsets inside a tile are the same for
// every tile, so that a tile costs a scalar base per tensor and no vector arithmetic.
__device__ inline unsigned lds_address(const void *p) {
    return __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(__attribute__((address_space(3))) const void *)p);
}
template <typename P> __device__ inline P *uniform(P *p) {
    const uint64_t x = (uint64_t)p;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x), hi = __builtin_amdgcn_readfirstlane((uint32_t)(x >> 32));
    return (P *)(((uint64_t)hi << 32) | lo);
}
__device__ inline void lds_dma(const char *base, unsigned lane_off, unsigned lds_byte) {
    asm volatile("s_mov_b32 m0, %1\n\t"
                 "s_nop 0\n\t"
                 "global_load_lds_dwordx4 %0, %2"
                 :
                 : "v"(lane_off), "s"(__builtin_amdgcn_readfirstlane(lds_byte)), "s"(uniform(base))
                 : "memory" SDPA_M0_CLOBBER);
}

// 4 bytes a lane: 64 consecutive words
__device__ inline void lds_dma_words(const void *base, int lane, unsigned lds_byte) {
    asm volatile("s_mov_b32 m0, %1\n\t"
                 "s_nop 0\n\t"
                 "global_load_lds_dword %0, %2"
                 :
                 : "v"(lane * 4), "s"(__builtin_amdgcn_readfirstlane(lds_byte)), "s"(uniform((const char *)base))
                 : "memory" SDPA_M0_CLOBBER);
}

// A tile of ROWS rows of a key list, staged by WAVES waves.  Rows behind the list's end are read as its last key (their weights are
// masked), so that nothing is read that no query of the workgroup sees.
// The waves take the tile's 1 KiB pieces in turn: with four waves a wave's pieces lie 4 KiB apart, where the swizzle (period 16
// rows) repeats, or nearly so -- kKinds lane offsets serve all of them, the rest of a piece's place is uniform.
template <typename T, int DP, int ROWS, int WAVES> struct Stager {
    using TL = Tile<T, DP>;
    static constexpr int kPieces = ROWS * TL::kRowBytes / 1024 / WAVES;       // pieces of a wave
    static constexpr int kKinds = TL::kRowBytes * 16 / 1024 / WAVES < 1 ? 1 : TL::kRowBytes * 16 / 1024 / WAVES;
    const char *base;                // row 0 of the head
    long token;                      // bytes between rows
    int dim;
    unsigned off[kKinds];            // lane offsets inside a tile
    unsigned has;                    // bit k: off[k] is a chunk of the row, not of its padding
    __device__ static int row(int wave, int lane, int k) { return (((wave + k * WAVES) * 1024 + lane * 16) / TL::kRowBytes); }
    __device__ static int source(int wave, int lane, int k) {                 // the chunk of its row a lane asks for
        return (((wave + k * WAVES) * 64 + lane) % TL::kChunks) ^ TL::swz(row(wave, lane, k));
    }
    __device__ void init(const void *p, long tok, int d, int wave, int lane) {
        base = uniform((const char *)p);
        token = tok * (long)sizeof(T);
        dim = d;
#pragma unroll
        for (int k = 0; k < kKinds; ++k) off[k] = (unsigned)(row(wave, lane, k) * (int)token) + 16u * (unsigned)source(wave, lane, k);
        has = 0;
#pragma unroll
        for (int k = 0; k < kKinds; ++k) has |= source(wave, lane, k) * Ops<T>::kVec < d ? 1u << k : 0u;
    }
    // asynchronous: 16-byte rows (a tile's offsets fit 32 bits).  -> true: exactly kPieces instructions are on their way
    __device__ bool dma(unsigned lds, int v0, const KeyList &l, int wave, int lane) const {
        const char *at = base + (long)l.key(v0) * token;
        lds += (unsigned)wave * 1024u;
        if (v0 + ROWS <= l.n && (v0 >= l.s || v0 + ROWS <= l.s)) {
            const long step = token * (kKinds * WAVES * 1024 / TL::kRowBytes);
            if (dim == DP) {
#pragma unroll
                for (int k = 0; k < kPieces; ++k) lds_dma(at + k / kKinds * step, off[k % kKinds], lds + k * WAVES * 1024u);
                return true;
            }
#pragma unroll
            for (int k = 0; k < kPieces; ++k)
                if ((has >> (k % kKinds)) & 1) lds_dma(at + k / kKinds * step, off[k % kKinds], lds + k * WAVES * 1024u);   // (the padding stays zero)
            return false;
        } else {
            const int ln = opaque(lane), split = v0 < l.s && l.s < l.n ? l.s : l.n;     // entries of either side: a base each
            const char *above = base + (long)l.key(split < l.n ? split : v0) * token;
#pragma unroll 1
            for (int k = 0; k < kPieces; ++k) {
                const int r = row(wave, ln, k), c = source(wave, ln, k), v = v0 + r < l.n ? v0 + r : l.n - 1;
                if (c * Ops<T>::kVec < dim) {
                    if (v < split) lds_dma(at, (unsigned)((v - v0) * (int)token) + 16u * (unsigned)c, lds + k * WAVES * 1024u);
                    else lds_dma(above, (unsigned)((v - split) * (int)token) + 16u * (unsigned)c, lds + k * WAVES * 1024u);
                }
            }
            return false;
        }
    }
    // element by element, for rows without 16-byte alignment
    __device__ void copy(char *tile, int v0, const KeyList &l, int wave, int lane) const {
#pragma unroll 4
        for (int k = 0; k < kPieces; ++k) {
            const int ln = opaque(lane), r = row(wave, ln, k), c = source(wave, ln, k), v = v0 + r < l.n ? v0 + r : l.n - 1;
            const T *src = reinterpret_cast<const T *>(base + (long)l.key(v) * token);
            *reinterpret_cast<u32x4 *>(tile + (wave + k * WAVES) * 1024 + ln * 16) = load_chunk(src, c * Ops<T>::kVec, dim, false);
        }
    }
};
// LDS tiles whose padding no DMA ever writes
__device__ inline void zero_lds(char *p, int bytes, int threads) {
    for (int i = threadIdx.x * 16; i < bytes; i += threads * 16) *reinterpret_cast<u32x4 *>(p + i) = u32x4{0, 0, 0, 0};
}
__device__ inline void dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
template <int N> __device__ inline void dma_wait_but() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

}  // namespace heads
}  // namespace sdpa
