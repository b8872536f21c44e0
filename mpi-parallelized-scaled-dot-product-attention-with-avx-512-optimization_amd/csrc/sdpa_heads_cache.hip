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

// exclusive prefix sum of `count` over the workgroup's threads.  `sums`: one word a wave.
__device__ inline int block_before(int count, int *sums) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int scan = count;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int up = __shfl_up(scan, d);
        if (lane >= d) scan += up;
    }
    if (lane == 63) sums[wave] = scan;
    __syncthreads();
    int before = scan - count;
#pragma unroll
    for (int w = 0; w < kSelectThreads / 64; ++w) before += w < wave ? sums[w] : 0;
    __syncthreads();
    return before;
}

// One workgroup per (sequence, key head).  The c-th greatest weight is found digit by digit (four passes of 8 bits over a
// histogram in LDS, integer counts only); then every thread numbers what stays of its own run of keys, behind two prefix sums over
// the threads.  The weights are read once, into LDS (LOCAL: up to kSelectLocal keys); 8192 keys of 128 heads take 19 us --
// reading them again in every pass took 26 us.
constexpr int kSelectLocal = 32768;
template <bool LOCAL>
__global__ __launch_bounds__(kSelectThreads) void select_kernel(EvictArgs a) {
    extern __shared__ float local[];
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
    for (int i = live + tid; i < a.budget; i += kSelectThreads) { kept[i] = -1; wo[i] = 0.f; }
    if (n <= a.budget) {
        for (int j = tid; j < n; j += kSelectThreads) { kept[j] = j; wo[j] = w[j]; }
        return;
    }
    if (LOCAL) {
#pragma unroll 8
        for (int j = tid; j < n; j += kSelectThreads) local[j] = w[j];
        __syncthreads();
    }
    auto weight = [&](int j) { return LOCAL ? local[j] : w[j]; };
    const int lo = a.sinks, hi = n - a.recent, want = a.budget - a.sinks - a.recent;
    uint32_t bar = 0xffffffffu;                       // weights above it stay, and the first `ties` equal to it (no weight has that key)
    int ties = 0;
    if (want > 0) {
        uint32_t prefix = 0;
        int left = want;                              // how many of the current candidates stay
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
#pragma unroll 4
            for (int j = lo + tid; j < hi; j += kSelectThreads) {
                const uint32_t key = order_key(weight(j));
                if (shift == 24 || (key >> ((shift + 8) & 31)) == prefix) atomicAdd(&hist[(key >> shift) & 255], 1);
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
        bar = prefix;
        ties = left;
    }
    // a thread's run of keys (an odd number of them: the threads' reads fall into different banks)
    const int run = ((n + kSelectThreads - 1) / kSelectThreads) | 1, j0 = min(tid * run, n), j1 = min(j0 + run, n);
    int equal = 0;
    for (int j = max(j0, lo); j < min(j1, hi); ++j) equal += order_key(weight(j)) == bar ? 1 : 0;
    equal = block_before(equal, sums);
    auto stays = [&](int j, int &rank) {              // `rank`: ties so far
        if (j < lo || j >= hi) return true;
        const uint32_t key = order_key(weight(j));
        return key > bar || (key == bar && rank++ < ties);
    };
    int count = 0, rank = equal;
    for (int j = j0; j < j1; ++j) count += stays(j, rank) ? 1 : 0;
    int at = block_before(count, sums);
    rank = equal;
    for (int j = j0; j < j1; ++j)
        if (stays(j, rank)) { kept[at] = j; wo[at] = weight(j); ++at; }
}

// The rows that stay, in pieces of one U: 4 pieces a thread.  K's workgroups come first, then V's.  At the rate of a copy: 4096 of 8192
// tokens of 16 sequences, 8 heads of 128 columns, bf16, 103 us, 537 MB = 5.2 TB/s.  Rows off 16 bytes move element by element: the call takes
// 305 us with 100 columns, 111 with 96 (fp32 250 and 173).
struct GatherSide { sdpa_tensor in, out; int pieces, blocks; };
template <typename U>
__global__ __launch_bounds__(kHeadsThreads) void gather_kernel(EvictArgs a, GatherSide k, GatherSide v) {
    int id = blockIdx.x;
    const int k_blocks = a.B * a.H * k.blocks;
    const bool is_v = id >= k_blocks;
    const GatherSide &g = is_v ? v : k;
    if (is_v) id -= k_blocks;
    const int part = id % g.blocks;
    id /= g.blocks;
    const int h = id % a.H, b = id / a.H;
    const int *kept = a.kept + ((long)b * a.H + h) * a.budget;
    const U *src = reinterpret_cast<const U *>((const char *)g.in.data + (b * g.in.batch + h * g.in.head) * a.elem);
    U *dst = reinterpret_cast<U *>((char *)g.out.data + (b * g.out.batch + h * g.out.head) * a.elem);
    const long in_row = g.in.token * a.elem / (long)sizeof(U), out_row = g.out.token * a.elem / (long)sizeof(U);
    U x[4];
    int slot[4], c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const long at = (long)part * (kHeadsThreads * 4) + i * kHeadsThreads + threadIdx.x;
        slot[i] = (int)(at / g.pieces);
        c[i] = (int)(at - (long)slot[i] * g.pieces);
        const int j = slot[i] < a.budget ? kept[slot[i]] : -1;
        x[i] = U{};
        if (j >= 0) x[i] = src[j * in_row + c[i]];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (slot[i] < a.budget) dst[slot[i] * out_row + c[i]] = x[i];
}

template <typename U> void gather(const EvictArgs &a, hipStream_t s) {
    auto side = [&](const sdpa_tensor &in, const sdpa_tensor &out, int dim) {
        GatherSide g = {in, out, dim * a.elem / (int)sizeof(U), 0};
        g.blocks = (int)(((long)a.budget * g.pieces + kHeadsThreads * 4 - 1) / (kHeadsThreads * 4));
        return g;
    };
    const GatherSide k = side(a.k, a.k_out, a.Dk), v = side(a.v, a.v_out, a.Dv);
    gather_kernel<U><<<a.B * a.H * (k.blocks + v.blocks), kHeadsThreads, 0, s>>>(a, k, v);
}

}  // namespace
}  // namespace heads

hipError_t launch_evict(const EvictArgs &a, hipStream_t s) {
    const int groups = a.B * a.H;
    if (a.Tk <= heads::kSelectLocal) {
        const size_t bytes = (size_t)a.Tk * 4;
        if (bytes > 32768) {                             // (an attribute of the device's function: not kept for the process)
            const hipError_t e = hipFuncSetAttribute((const void *)heads::select_kernel<true>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                                     heads::kSelectLocal * 4);
            if (e != hipSuccess) return e;
        }
        heads::select_kernel<true><<<groups, heads::kSelectThreads, bytes, s>>>(a);
    } else {
        heads::select_kernel<false><<<groups, heads::kSelectThreads, 0, s>>>(a);
    }
    if (a.budget == 0) return hipGetLastError();
    if (a.vec) heads::gather<heads::u32x4>(a, s);
    else if (a.elem == 4) heads::gather<uint32_t>(a, s);
    else heads::gather<uint16_t>(a, s);
    return hipGetLastError();
}

}  // namespace sdpa
