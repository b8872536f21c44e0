// sdpa_heads_cache.hip -- eviction from a cache by accumulated weight: which keys stay, and their move to the front.
#include "sdpa_heads_device.h"

namespace sdpa {
namespace heads {
namespace {

constexpr int kSelectThreads = 1024;

// A weight as a number whose unsigned order is the weights': sign and magnitude to two's order; -0 as 0; NaN below everything.
__device__ inline uint32_t order_key(float w) {
    const uint32_t u = __float_as_uint(w + 0.f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return 0;
    return u >> 31 ? ~u : u | 0x80000000u;
}

// exclusive prefix count of `flag` over the workgroup's threads; `total` = all of them.  `sums`: one word a wave.
__device__ inline int block_rank(bool flag, int *sums, int *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint64_t mask = __ballot(flag);
    if (lane == 0) sums[wave] = __popcll(mask);
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kSelectThreads / 64; ++w) {
        const int c = sums[w];
        before += w < wave ? c : 0;
        all += c;
    }
    __syncthreads();
    *total = all;
    return before + __popcll(mask & ((1ull << lane) - 1));
}

// One workgroup per (sequence, key head).  The c-th greatest weight is found digit by digit (four passes of 8 bits over a
// histogram in LDS, integer counts only); then one ordered pass numbers what stays.
__global__ __launch_bounds__(kSelectThreads) void select_kernel(EvictArgs a) {
    __shared__ int hist[256];
    __shared__ int sums[kSelectThreads / 64];
    __shared__ uint32_t s_prefix;
    __shared__ int s_left;
    const int tid = threadIdx.x, h = blockIdx.x % a.H, b = blockIdx.x / a.H;
    const int n = clamp_len(a.lens, b, a.Tk), live = n < a.budget ? n : a.budget;
    const float *w = a.w_in + b * a.wi_batch + h * a.wi_head;
    float *wo = a.w_out + b * a.wo_batch + h * a.wo_head;
    int *kept = a.kept + ((long)b * a.H + h) * a.budget;
    if (h == 0 && tid == 0) a.lens_out[b] = live;
    const int lo = a.sinks, hi = n - a.recent;
    uint32_t bar = 0;                                 // weights above it stay, and the first `ties` equal to it
    int ties = 1 << 30;
    if (n > a.budget) {
        const int want = a.budget - a.sinks - a.recent;
        uint32_t prefix = 0;
        int left = want;                              // how many of the current candidates stay
        for (int shift = 24; shift >= 0 && left > 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (int j = lo + tid; j < hi; j += kSelectThreads) {
                const uint32_t key = order_key(w[j]);
                if (shift == 24 || (key >> (shift + 8)) == prefix) atomicAdd(&hist[(key >> shift) & 255], 1);
            }
            __syncthreads();
            if (tid < 64) {                           // the digit in which the left-th greatest candidate lies
                int c[4], above = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) { c[i] = hist[255 - 4 * tid - i]; above += c[i]; }
                int scan = above;
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) {
                    const int up = __shfl_up(scan, d);
                    if (tid >= d) scan += up;
                }
                int before = scan - above;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (before < left && before + c[i] >= left) {
                        s_prefix = (prefix << 8) | (uint32_t)(255 - 4 * tid - i);
                        s_left = left - before;
                    }
                    before += c[i];
                }
            }
            __syncthreads();
            prefix = s_prefix;
            left = s_left;
        }
        if (want == 0) { bar = 0xffffffffu; ties = 0; }          // (no weight has that key)
        else { bar = prefix; ties = left; }
    }
    int out = 0, equal = 0;
    for (int base = 0; base < n; base += kSelectThreads) {
        const int j = base + tid;
        const float x = j < n ? w[j] : 0.f;
        bool stays = j < n;
        if (n > a.budget) {
            const bool fixed = j < lo || j >= hi;
            const uint32_t key = order_key(x);
            const bool tie = j < n && !fixed && key == bar;
            int total;
            const int rank = block_rank(tie, sums, &total);
            stays = j < n && (fixed || key > bar || (tie && equal + rank < ties));
            equal += total;
        }
        int total;
        const int at = out + block_rank(stays, sums, &total);
        if (stays) { kept[at] = j; wo[at] = x; }
        out += total;
    }
    for (int i = live + tid; i < a.budget; i += kSelectThreads) { kept[i] = -1; wo[i] = 0.f; }
}

// `UNIT`-byte pieces of rows: a thread moves one piece of K or V
template <typename U>
__global__ __launch_bounds__(kHeadsThreads) void gather_kernel(EvictArgs a, sdpa_tensor in, sdpa_tensor out, int pieces, int blocks) {
    int id = blockIdx.x;
    const int part = id % blocks;
    id /= blocks;
    const int h = id % a.H, b = id / a.H;
    const int *kept = a.kept + ((long)b * a.H + h) * a.budget;
    const U *src = reinterpret_cast<const U *>((const char *)in.data + (b * in.batch + h * in.head) * a.elem);
    U *dst = reinterpret_cast<U *>((char *)out.data + (b * out.batch + h * out.head) * a.elem);
    const long in_row = in.token * a.elem / (long)sizeof(U), out_row = out.token * a.elem / (long)sizeof(U);
    const int per = kHeadsThreads * 4;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const long i = (long)part * per + k * kHeadsThreads + threadIdx.x;
        const int slot = (int)(i / pieces), c = (int)(i - (long)slot * pieces);
        if (slot >= a.budget) return;
        const int j = kept[slot];
        U v = {};
        if (j >= 0) v = src[j * in_row + c];
        dst[slot * out_row + c] = v;
    }
}

template <typename U>
void gather(const EvictArgs &a, const sdpa_tensor &in, const sdpa_tensor &out, int dim, hipStream_t s) {
    const int pieces = dim * a.elem / (int)sizeof(U);
    const int blocks = (int)(((long)a.budget * pieces + kHeadsThreads * 4 - 1) / (kHeadsThreads * 4));
    gather_kernel<U><<<a.B * a.H * blocks, kHeadsThreads, 0, s>>>(a, in, out, pieces, blocks);
}

void gather_any(const EvictArgs &a, const sdpa_tensor &in, const sdpa_tensor &out, int dim, int vec, hipStream_t s) {
    if (vec) gather<u32x4>(a, in, out, dim, s);
    else if (a.elem == 4) gather<uint32_t>(a, in, out, dim, s);
    else gather<uint16_t>(a, in, out, dim, s);
}

}  // namespace
}  // namespace heads

hipError_t launch_evict(const EvictArgs &a, hipStream_t s) {
    heads::select_kernel<<<a.B * a.H, heads::kSelectThreads, 0, s>>>(a);
    if (a.budget == 0) return hipGetLastError();
    heads::gather_any(a, a.k, a.k_out, a.Dk, a.vec_k, s);
    heads::gather_any(a, a.v, a.v_out, a.Dv, a.vec_v, s);
    return hipGetLastError();
}

}  // namespace sdpa
