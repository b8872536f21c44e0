// sdpa_heads.h -- the batched attention operators: what the C ABI hands to the launchers, and the rules both share.
// Internal; the public interface is include/sdpa_hip.h (struct sdpa_heads).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>

#include "../../include/sdpa_hip.h"

namespace sdpa {

constexpr int kHeadDimMax = 256;      // the widest head whose O^T columns stay in registers beside its Q fragments
constexpr int kFewRows    = 32;       // query rows of one MFMA column block: up to here waves split the KEYS, beyond the rows

// padded head width of the kernels' tiles
inline int heads_pad(int dk, int dv) {
    const int d = dk > dv ? dk : dv;
    return d <= 64 ? 64 : d <= 128 ? 128 : 256;
}
inline int elem_bytes(int dtype) { return dtype == SDPA_BF16 ? 2 : 4; }

// 16-byte accesses hold for a tensor whose base, strides and row length are multiples of 16 bytes (and whose tiles of up to 128
// rows fit 32-bit offsets)
inline bool rows_vec(const sdpa_tensor &t, int dim, int dtype) {
    const long e = elem_bytes(dtype), bad = (t.batch * e) | (t.token * e) | (t.head * e) | (dim * e);
    return ((bad | (long)(size_t)t.data) & 15) == 0 && t.token < (1 << 21);
}

// the few-rows kernel: bytes of a 32-key K and V tile, and the waves of its wide form (128 KiB of LDS)
constexpr int few_pair_bytes(int pad, int elem) { return 2 * 32 * pad * elem; }
constexpr int few_wide_waves(int pad, int elem) { return 131072 / few_pair_bytes(pad, elem) < 8 ? 131072 / few_pair_bytes(pad, elem) : 8; }

// One launch over one set of keys: its queries, where its rows go, and what they may see.
struct AttendArgs {
    sdpa_tensor q, k, v, out;
    float *lse;                       // [B][Hq][Tq]
    const int *q_lens, *kv_lens;      // [B] or null
    float *part;                      // [slots][B*Tq*Hq][Dv] un-normalised rows (null: the launch writes out / lse itself)
    float2 *stat;                     // [slots][B*Tq*Hq] (reference exponent, sum)
    float *scores;                    // [B][Hkv][Tq * G][score_ld] raw scores for the weights (launches over few rows; may be null)
    long score_ld;
    int slot0, splits;                // this launch's slots
    int B, Tq, Tk, Hq, Hkv, Dk, Dv;
    int window, sinks;
    int wide;                         // few rows: one workgroup of more waves to a head, no splits
    int shared;                       // 1 = one set of keys for the whole batch, all of them visible (a prefix)
    int vec, vec_out;                 // 16-byte loads of q, k, v / whole 4-element stores of out
    int q_sign;                       // the softmax scale's sign: applied to the queries
    float scale_log2;                 // its magnitude * log2(e) (1 for a scale of 0): scores are kept in the exp2 domain
};

struct BackwardArgs {
    sdpa_tensor q, k, v, out, dout, dq, dk, dv;
    const float *lse;
    float *stats;                     // [2][B * Hkv][stat_rows]: lse (exp2 domain) and -sum dO * O of the rows, in the keys kernel's order
    long stat_rows, stat_stride;      // (a multiple of 64; the second array's offset)
    float *part;                      // partial dK | dV rows of the key blocks whose queries several workgroups share
    const int *q_lens, *kv_lens;
    int B, Tq, Tk, Hq, Hkv, Dk, Dv;
    int window, sinks;
    int chunks;                       // workgroups that share a key block's rows
    int sink_blocks, tail_chunks;     // key blocks with sink keys, and the workgroups for their rows behind the window
    int vec, vec_out, dma;            // 16-byte loads / stores; tiles by DMA
    float scale, scale_log2;
};

// attention_scored: the weights every key was given, from the scores that were kept or from the products once more
struct WeightArgs {
    sdpa_tensor q, k;
    const float *lse, *w_in;
    float *w_out;
    const float *scores;
    const float2 *stat;               // the slots of the rows (null: lse holds)
    long score_ld;
    int slots;
    long wi_batch, wi_head, wo_batch, wo_head;
    const int *q_lens, *kv_lens;
    int B, Tq, Tk, Hq, Hkv, Dk, vec;
    float scale_log2;
};

struct EvictArgs {
    sdpa_tensor k, v, k_out, v_out;
    const float *w_in;
    float *w_out;
    long wi_batch, wi_head, wo_batch, wo_head;
    const int *lens;
    int *lens_out, *kept;
    int B, Tk, H, Dk, Dv, budget, sinks, recent, elem;
    int vec;                          // rows in 16-byte pieces
};

hipError_t launch_attend(const AttendArgs &a, int dtype, hipStream_t s);
hipError_t launch_combine(const AttendArgs &a, int slots, int dtype, hipStream_t s);
// the same and, in the same launch, w_out from the scores kept by launch_attend
hipError_t launch_combine_scored(const AttendArgs &a, const WeightArgs &w, int slots, int dtype, hipStream_t s);
hipError_t launch_attend_backward(const BackwardArgs &a, int dtype, hipStream_t s);
hipError_t launch_weights(const WeightArgs &a, int dtype, hipStream_t s);
hipError_t launch_evict(const EvictArgs &a, hipStream_t s);

constexpr int kBwdKeys = 64;          // keys of a dK / dV workgroup

}  // namespace sdpa
