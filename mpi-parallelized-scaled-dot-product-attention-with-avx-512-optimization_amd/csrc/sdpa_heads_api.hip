// sdpa_heads_api.hip -- the C ABI of the batched attention operators: argument checks, work plans, scratch.
#include "sdpa_errors.h"
#include "sdpa_heads.h"

#include <limits.h>
#include <math.h>
#include <stdint.h>

namespace {

using namespace sdpa;

constexpr int kMaxTokens = 1 << 30;
constexpr int kMaxSplits = 64;
constexpr float kMaxScale = 0x1p127f;     // times log2(e) it is finite still: a larger one would make NaN of scores of 0
constexpr double kMaxRows = (1 << 24) - 1, kMaxGroups = (1 << 24) - 1;

bool bad_tensor(const sdpa_tensor &t, bool needed) {
    return (needed && !t.data) || t.batch < 0 || t.token < 0 || t.head < 0;
}
// an output that repeats elements (a stride of 0) would be written by several workgroups
bool repeats(const sdpa_tensor &t, int batch, int tokens, int heads) {
    return (batch > 1 && t.batch == 0) || (tokens > 1 && t.token == 0) || (heads > 1 && t.head == 0);
}

bool repeats_weights(const sdpa_heads *a) {
    return (a->batch > 1 && a->weights_out_batch == 0) || (a->kv_heads > 1 && a->weights_out_head == 0);
}

long ceil_div(long a, long b) { return (a + b - 1) / b; }

int check_shape(const sdpa_heads *a) {
    if (!a || a->size != sizeof(sdpa_heads)) return SDPA_EINVAL;
    if (a->dtype != SDPA_F32 && a->dtype != SDPA_BF16) return SDPA_EINVAL;
    if (a->batch < 0 || a->q_tokens < 0 || a->kv_tokens < 0 || a->kv_heads < 1 || a->dk < 1 || a->dv < 1) return SDPA_EINVAL;
    if (a->dk > kHeadDimMax || a->dv > kHeadDimMax) return SDPA_EUNSUP;
    if (a->q_tokens > kMaxTokens || a->kv_tokens > kMaxTokens) return SDPA_EUNSUP;
    return SDPA_OK;
}

int check_attention(const sdpa_heads *a) {
    SDPA_TRY(check_shape(a));
    if (a->q_heads < 1 || a->q_heads % a->kv_heads != 0) return SDPA_EINVAL;
    if (a->window < 0 || a->sinks < 0 || a->prefix_tokens < 0) return SDPA_EINVAL;
    if (!(fabsf(a->scale) <= kMaxScale)) return SDPA_EINVAL;
    if (a->prefix_tokens > kMaxTokens) return SDPA_EUNSUP;
    // a launch has less than 2^32 threads: 256 for each 128 keys or rows of a head, and for each row of a join.  Of the forward forms only
    // few rows are split and joined, and those beside a prefix, whose rows are one tile list for the batch.
    const double groups = (double)a->batch * a->kv_heads, rows = (double)a->q_tokens * (a->q_heads / a->kv_heads);
    if (rows > kMaxRows || groups * (ceil_div(a->kv_tokens, 128) + 1) > kMaxGroups || groups * (rows / 128 + 1) > kMaxGroups ||
        (a->prefix_tokens > 0 && groups * rows > kMaxRows))
        return SDPA_EUNSUP;
    return SDPA_OK;
}

bool empty(const sdpa_heads *a) { return a->batch == 0 || a->q_tokens == 0; }

// How many workgroups share the keys of a row tile.  A launch wants about two workgroups on each of the 256 CUs; a split costs a
// partial row (4 * dv + 8 bytes written and read) per query row and needs keys enough to be worth its start: one 32-key tile
// for each of its waves where they take the keys in turn, a tile of 64 where they share it.
int pick_splits(int dtype, long groups, long rows, long keys) {
    const long tiles = rows <= kFewRows ? 1 : ceil_div(rows, 128);
    const long have = groups * tiles;
    // (few rows: measured flat between 512 and 768 workgroups.  Many rows: never a second, mostly empty round; fp32 workgroups are bound by
    // their matrix instructions and gain nothing from a neighbour on their CU.)
    long want = rows <= kFewRows ? ceil_div(512, have < 1 ? 1 : have) : (dtype == SDPA_BF16 ? 512 : 256) / (have < 1 ? 1 : have);
    const long most = ceil_div(keys, rows <= kFewRows ? 128 : 64);
    if (want > most) want = most;
    if (want > kMaxSplits) want = kMaxSplits;
    return want < 1 ? 1 : (int)want;
}

AttendArgs attend_args(const sdpa_heads *a) {
    AttendArgs x = {};
    x.q = a->q; x.k = a->k; x.v = a->v; x.out = a->out;
    x.lse = a->lse; x.q_lens = a->q_lens; x.kv_lens = a->kv_lens;
    x.B = a->batch; x.Tq = a->q_tokens; x.Tk = a->kv_tokens; x.Hq = a->q_heads; x.Hkv = a->kv_heads; x.Dk = a->dk; x.Dv = a->dv;
    x.window = a->window < kMaxTokens ? a->window : kMaxTokens;
    x.sinks = a->sinks;
    x.splits = 1;
    x.vec = rows_vec(a->q, a->dk, a->dtype) && rows_vec(a->k, a->dk, a->dtype) && rows_vec(a->v, a->dv, a->dtype);
    x.vec_out = rows_vec(a->out, a->dv, a->dtype);
    x.q_sign = a->scale > 0.f ? 1 : a->scale < 0.f ? -1 : 0;
    x.scale_log2 = a->scale == 0.f ? 1.f : fabsf(a->scale) * 1.44269504088896341f;
    return x;
}

// keys a tile of rows may see at most
long keys_seen(const sdpa_heads *a, long rows) {
    const long G = a->q_heads / a->kv_heads, tile = rows <= kFewRows ? rows : 128;
    const long w = (long)a->window + ceil_div(tile, G) + a->sinks;
    return w < a->kv_tokens ? w : a->kv_tokens;
}

// A call so small that one workgroup a head does it: at most four tiles of 32 keys for each of its waves, and a CU for every head.  (One
// launch instead of two.)
bool one_workgroup(const sdpa_heads *a, long groups, long rows, long keys) {
    return rows <= kFewRows && groups <= 256 && ceil_div(keys, 32) <= 4 * few_wide_waves(heads_pad(a->dk, a->dv), elem_bytes(a->dtype));
}

struct Slots {
    bool wide;                    // few rows: the form with one workgroup a head
    int own, prefix;              // slots of the sequences' own keys and of the prefix
    long rows, part, bytes;       // bytes of the slots, and of everything
    long score_ld;                // kept scores (attention_scored over few rows): their row, 0 = none
    void size(const sdpa_heads *a, bool scored) {
        rows = (long)a->batch * a->q_tokens * a->q_heads;
        const int n = own + prefix;
        part = n > 1 ? ((n * rows * 8 + 15) / 16 * 16 + n * rows * (long)a->dv * 4 + 15) / 16 * 16 : 0;
        score_ld = scored && (long)a->q_tokens * (a->q_heads / a->kv_heads) <= kFewRows ? ceil_div(a->kv_tokens, 32) * 32 : 0;
        bytes = part + rows * score_ld * 4;
    }
};

Slots plan_window(const sdpa_heads *a, bool scored) {
    Slots s = {};
    const long rows = (long)a->q_tokens * (a->q_heads / a->kv_heads);
    const long groups = (long)a->batch * a->kv_heads, keys = keys_seen(a, rows);
    if (one_workgroup(a, groups, rows, keys)) { s.wide = true; s.own = 1; }
    else s.own = pick_splits(a->dtype, groups, rows, keys);
    s.size(a, scored);
    return s;
}

Slots plan_prefix(const sdpa_heads *a) {
    Slots s = {};
    const long rows = (long)a->q_tokens * (a->q_heads / a->kv_heads);
    s.own = pick_splits(a->dtype, (long)a->batch * a->kv_heads, rows, a->kv_tokens);
    s.prefix = a->prefix_tokens > 0 ? pick_splits(a->dtype, a->kv_heads, rows * a->batch, a->prefix_tokens) : 0;
    s.size(a, false);
    return s;
}

void carve(AttendArgs &x, const Slots &s, void *workspace) {
    if (s.own + s.prefix <= 1) return;
    x.stat = (float2 *)workspace;
    const size_t stat = ((size_t)(s.own + s.prefix) * s.rows * 8 + 15) / 16 * 16;
    x.part = (float *)((char *)workspace + stat);
}

int check_scratch(long need, const void *workspace, size_t bytes) {
    if (need > 0 && (!workspace || bytes < (size_t)need || ((uintptr_t)workspace & 15) != 0)) return SDPA_EINVAL;
    return SDPA_OK;
}

int check_forward(const sdpa_heads *a) {
    SDPA_TRY(check_attention(a));
    if (empty(a)) return SDPA_OK;
    if (bad_tensor(a->q, true) || bad_tensor(a->k, a->kv_tokens > 0) || bad_tensor(a->v, a->kv_tokens > 0) ||
        bad_tensor(a->out, true) || !a->lse)
        return SDPA_EINVAL;
    if (repeats(a->out, a->batch, a->q_tokens, a->q_heads)) return SDPA_EINVAL;
    return SDPA_OK;
}

// splits of a launch over one set of keys, then the join
int run_own(const sdpa_heads *a, const Slots &s, void *workspace, hipStream_t st) {
    AttendArgs x = attend_args(a);
    x.splits = s.own;
    x.wide = s.wide;
    carve(x, s, workspace);
    HIP_TRY(launch_attend(x, a->dtype, st));
    if (x.part) HIP_TRY(launch_combine(x, s.own, a->dtype, st));
    return SDPA_OK;
}

struct BackwardPlan { int chunks, sink_blocks, tail_chunks; long stat_rows, stats, bytes; double grid; };

// A key block's workgroup walks the rows that see it by the window, about (64 + window) tokens' heads; several share them while the launch
// has fewer workgroups than the chip has CUs.  A block with sink keys is seen by every row behind: its tail goes to short workgroups
// of their own, launched last (one walk in a row's length would outlast all others).
BackwardPlan plan_backward(const sdpa_heads *a) {
    BackwardPlan p = {};
    const long G = a->q_heads / a->kv_heads, groups = (long)a->batch * a->kv_heads, blocks = ceil_div(a->kv_tokens, kBwdKeys);
    const long sinks = a->sinks < a->kv_tokens ? a->sinks : a->kv_tokens, reach = (long)a->window + kBwdKeys;
    const long walk = (reach < a->q_tokens ? reach : a->q_tokens) * G, tail = reach < a->q_tokens ? (a->q_tokens - reach) * G : 0;
    long chunks = groups * blocks < 256 ? ceil_div(256, groups * blocks < 1 ? 1 : groups * blocks) : 1;
    if (chunks > ceil_div(walk, 128)) chunks = ceil_div(walk, 128);
    if (chunks > kMaxSplits) chunks = kMaxSplits;
    p.chunks = chunks < 1 ? 1 : (int)chunks;
    p.sink_blocks = (int)ceil_div(sinks, kBwdKeys);
    const long piece = walk / (4 * p.chunks) > 128 ? walk / (4 * p.chunks) : 128;
    const long tails = ceil_div(tail, piece);
    // Each of them has a slot in the scratch, so there are as many as fill the chip twice, or an eighth of the key blocks (a quarter of the
    // bytes of bf16 gradients), and where that leaves less than two to a block there is no need for them: so many long walks fill the chip
    // by themselves.
    const long busy = groups * blocks / 8 > 512 ? groups * blocks / 8 : 512, most = groups * p.sink_blocks < 1 ? 0 : busy / (groups * p.sink_blocks);
    p.tail_chunks = most < 2 ? 0 : (int)(tails < most ? tails < kMaxSplits ? tails : kMaxSplits : most < kMaxSplits ? most : kMaxSplits);
    // the largest launch, the join's 16 workgroups of a block among them (counted for every sink block with a tail, so that what is refused goes
    // by the sizes alone and not by the plan)
    const long joined = p.chunks > 1 ? blocks : tail > 0 ? p.sink_blocks : 0;
    p.grid = (double)groups * (blocks * p.chunks + p.sink_blocks * p.tail_chunks);
    if ((double)groups * joined * (kBwdKeys / 4) > p.grid) p.grid = (double)groups * joined * (kBwdKeys / 4);
    const long slots = p.chunks > 1 ? blocks * p.chunks + p.sink_blocks * p.tail_chunks :
                       p.tail_chunks > 0 ? p.sink_blocks * (1 + p.tail_chunks) : 0;
    // rows of a head: blocks of 32, whole tokens to a block (or, of larger groups, blocks to a token), in pairs
    const long row_blocks = G <= 32 ? ceil_div(a->q_tokens, 32 / G) : a->q_tokens * ceil_div(G, 32);
    p.stat_rows = ceil_div(row_blocks, 2) * 64;
    p.stats = 2 * groups * p.stat_rows * 4;
    p.bytes = p.stats + groups * slots * kBwdKeys * (a->dk + a->dv) * 4 + 16;
    return p;
}

// the plan of a call, or why there is none (for the call and for the question of its scratch)
int plan_backward(const sdpa_heads *a, BackwardPlan &p) {
    p = plan_backward(a);
    return p.grid > kMaxGroups ? SDPA_EUNSUP : SDPA_OK;
}

int check_evict(const sdpa_heads *a) {
    SDPA_TRY(check_shape(a));
    if (a->budget < 0 || a->sinks < 0 || a->recent < 0 || (long)a->sinks + a->recent > a->budget) return SDPA_EINVAL;
    if (a->budget > kMaxTokens) return SDPA_EUNSUP;
    if (a->batch == 0) return SDPA_OK;
    const bool in = a->kv_tokens > 0, out = a->budget > 0;
    if (bad_tensor(a->k, in) || bad_tensor(a->v, in) || bad_tensor(a->k_out, out) || bad_tensor(a->v_out, out))
        return SDPA_EINVAL;
    if ((in && !a->weights) || (out && (!a->weights_out || !a->kept)) || !a->lens_out) return SDPA_EINVAL;
    if (a->weights_batch < 0 || a->weights_head < 0 || a->weights_out_batch < 0 || a->weights_out_head < 0) return SDPA_EINVAL;
    if (out && repeats_weights(a)) return SDPA_EINVAL;
    // lengths and weights are read by workgroups that others' results of these would overtake
    const uintptr_t n_in = (uintptr_t)a->kv_lens, n_out = (uintptr_t)a->lens_out, n_bytes = (uintptr_t)a->batch * sizeof(int);
    if ((n_in && n_out < n_in + n_bytes && n_in < n_out + n_bytes) || (in && out && a->weights_out == a->weights)) return SDPA_EINVAL;
    if (repeats(a->k_out, a->batch, a->budget, a->kv_heads) || repeats(a->v_out, a->batch, a->budget, a->kv_heads))
        return SDPA_EINVAL;
    // (a workgroup moves 1024 pieces of at least one element, and one of 1024 threads selects for a head)
    const double units = (double)a->budget * (a->dk + a->dv), groups = (double)a->batch * a->kv_heads;
    if (groups * (units / 1024 + 2) > kMaxGroups || groups > kMaxGroups / 4) return SDPA_EUNSUP;
    return SDPA_OK;
}

}  // namespace

extern "C" {

long sdpa_dev_heads_workspace(int op, const struct sdpa_heads *a) {
    if (op < SDPA_OP_WINDOW || op > SDPA_OP_EVICT) return SDPA_EINVAL;
    if (op == SDPA_OP_EVICT) {
        const int c = check_evict(a);
        return c != SDPA_OK ? c : 0;
    }
    int c = check_attention(a);
    if (c != SDPA_OK) return c;
    if (op == SDPA_OP_WINDOW_BACKWARD) {
        BackwardPlan p;
        c = plan_backward(a, p);
        return c != SDPA_OK ? c : p.bytes;
    }
    if (empty(a)) return 0;
    sdpa_heads x = *a;
    if (op == SDPA_OP_PREFIX || op == SDPA_OP_SCORED) { x.window = kMaxTokens; x.sinks = 0; }
    return op == SDPA_OP_PREFIX ? plan_prefix(&x).bytes : plan_window(&x, op == SDPA_OP_SCORED).bytes;
}

int sdpa_dev_attention_window(const struct sdpa_heads *a, void *workspace, size_t workspace_bytes, void *stream) {
    SDPA_TRY(check_forward(a));
    if (empty(a)) return SDPA_OK;
    const Slots s = plan_window(a, false);
    SDPA_TRY(check_scratch(s.bytes, workspace, workspace_bytes));
    SDPA_TRY(require_device());
    return run_own(a, s, workspace, (hipStream_t)stream);
}

int sdpa_dev_attention_window_backward(const struct sdpa_heads *a, void *workspace, size_t workspace_bytes, void *stream) {
    SDPA_TRY(check_attention(a));
    if (a->batch == 0) return SDPA_OK;
    const bool q = a->q_tokens > 0, k = a->kv_tokens > 0;
    if (bad_tensor(a->q, q) || bad_tensor(a->out, q) || bad_tensor(a->dout, q) || bad_tensor(a->dq, q) ||
        bad_tensor(a->k, k) || bad_tensor(a->v, k) || bad_tensor(a->dk_out, k) || bad_tensor(a->dv_out, k) || (q && !a->lse))
        return SDPA_EINVAL;
    if (repeats(a->dq, a->batch, a->q_tokens, a->q_heads) || repeats(a->dk_out, a->batch, a->kv_tokens, a->kv_heads) ||
        repeats(a->dv_out, a->batch, a->kv_tokens, a->kv_heads))
        return SDPA_EINVAL;
    BackwardPlan p;
    SDPA_TRY(plan_backward(a, p));
    SDPA_TRY(check_scratch(p.bytes, workspace, workspace_bytes));
    SDPA_TRY(require_device());
    BackwardArgs x = {};
    x.q = a->q; x.k = a->k; x.v = a->v; x.out = a->out; x.dout = a->dout; x.dq = a->dq; x.dk = a->dk_out; x.dv = a->dv_out;
    x.lse = a->lse; x.q_lens = a->q_lens; x.kv_lens = a->kv_lens;
    x.stats = (float *)workspace;
    x.stat_rows = p.stat_rows;
    x.stat_stride = (long)a->batch * a->kv_heads * p.stat_rows;
    x.part = (float *)((char *)workspace + p.stats);
    x.B = a->batch; x.Tq = a->q_tokens; x.Tk = a->kv_tokens; x.Hq = a->q_heads; x.Hkv = a->kv_heads; x.Dk = a->dk; x.Dv = a->dv;
    x.window = a->window < kMaxTokens ? a->window : kMaxTokens;
    x.sinks = a->sinks;
    x.chunks = p.chunks; x.sink_blocks = p.sink_blocks; x.tail_chunks = p.tail_chunks;
    x.vec = rows_vec(a->q, a->dk, a->dtype) && rows_vec(a->k, a->dk, a->dtype) && rows_vec(a->v, a->dv, a->dtype) &&
            rows_vec(a->out, a->dv, a->dtype) && rows_vec(a->dout, a->dv, a->dtype);
    // a tile of 64 rows: two blocks of 32 / G tokens' heads, at 32-bit offsets
    const long G = a->q_heads / a->kv_heads, e = elem_bytes(a->dtype);
    x.dma = x.vec && G <= 32 && (G * a->q.head + 64 / G * a->q.token) * e < INT_MAX / 2 && (G * a->dout.head + 64 / G * a->dout.token) * e < INT_MAX / 2;
    x.vec_out = rows_vec(a->dq, a->dk, a->dtype) && rows_vec(a->dk_out, a->dk, a->dtype) && rows_vec(a->dv_out, a->dv, a->dtype);
    x.scale = a->scale;
    x.scale_log2 = a->scale * 1.44269504088896341f;
    HIP_TRY(launch_attend_backward(x, a->dtype, (hipStream_t)stream));
    return SDPA_OK;
}

int sdpa_dev_attention_prefix(const struct sdpa_heads *a, void *workspace, size_t workspace_bytes, void *stream) {
    SDPA_TRY(check_forward(a));
    if (a->prefix_tokens > 0 && (bad_tensor(a->k_prefix, true) || bad_tensor(a->v_prefix, true))) return SDPA_EINVAL;
    if (empty(a)) return SDPA_OK;
    sdpa_heads own = *a;
    own.window = kMaxTokens;
    own.sinks = 0;
    const Slots s = plan_prefix(&own);
    SDPA_TRY(check_scratch(s.bytes, workspace, workspace_bytes));
    SDPA_TRY(require_device());
    if (s.prefix == 0) return run_own(&own, s, workspace, (hipStream_t)stream);
    AttendArgs x = attend_args(&own);
    x.splits = s.own;
    carve(x, s, workspace);
    HIP_TRY(launch_attend(x, a->dtype, (hipStream_t)stream));
    AttendArgs p = x;
    p.k = a->k_prefix; p.v = a->v_prefix;
    p.Tk = a->prefix_tokens;
    p.kv_lens = nullptr;
    p.shared = 1;
    p.slot0 = s.own;
    p.splits = s.prefix;
    p.vec = rows_vec(a->q, a->dk, a->dtype) && rows_vec(a->k_prefix, a->dk, a->dtype) && rows_vec(a->v_prefix, a->dv, a->dtype);
    HIP_TRY(launch_attend(p, a->dtype, (hipStream_t)stream));
    HIP_TRY(launch_combine(x, s.own + s.prefix, a->dtype, (hipStream_t)stream));
    return SDPA_OK;
}

int sdpa_dev_attention_scored(const struct sdpa_heads *a, void *workspace, size_t workspace_bytes, void *stream) {
    SDPA_TRY(check_forward(a));
    if (a->batch == 0) return SDPA_OK;
    if (a->kv_tokens > 0 && (!a->weights || !a->weights_out)) return SDPA_EINVAL;
    if (a->weights_batch < 0 || a->weights_head < 0 || a->weights_out_batch < 0 || a->weights_out_head < 0) return SDPA_EINVAL;
    if (a->kv_tokens > 0 && repeats_weights(a)) return SDPA_EINVAL;
    sdpa_heads x = *a;
    x.window = kMaxTokens;
    x.sinks = 0;
    Slots s = {};
    if (!empty(a)) {
        s = plan_window(&x, true);
        SDPA_TRY(check_scratch(s.bytes, workspace, workspace_bytes));
    }
    SDPA_TRY(require_device());
    WeightArgs w = {};
    w.q = a->q; w.k = a->k; w.lse = a->lse; w.w_in = a->weights; w.w_out = a->weights_out;
    w.wi_batch = a->weights_batch; w.wi_head = a->weights_head; w.wo_batch = a->weights_out_batch; w.wo_head = a->weights_out_head;
    w.q_lens = a->q_lens; w.kv_lens = a->kv_lens;
    w.B = a->batch; w.Tq = a->q_tokens; w.Tk = a->kv_tokens; w.Hq = a->q_heads; w.Hkv = a->kv_heads; w.Dk = a->dk;
    w.vec = rows_vec(a->q, a->dk, a->dtype) && rows_vec(a->k, a->dk, a->dtype);
    w.scale_log2 = a->scale * 1.44269504088896341f;
    if (!empty(a) && s.score_ld > 0) {                   // (over few rows) the scores are kept, and the weights come with the join
        AttendArgs f = attend_args(&x);
        f.splits = s.own;
        f.wide = s.wide;
        carve(f, s, workspace);
        f.scores = (float *)((char *)workspace + s.part);
        f.score_ld = s.score_ld;
        HIP_TRY(launch_attend(f, a->dtype, (hipStream_t)stream));
        w.scores = f.scores; w.score_ld = s.score_ld; w.stat = f.stat; w.slots = s.own;
        w.scale_log2 = f.scale_log2;                     // (their queries have the scale's sign already)
        HIP_TRY(launch_combine_scored(f, w, s.own, a->dtype, (hipStream_t)stream));
        return SDPA_OK;
    }
    if (!empty(a)) SDPA_TRY(run_own(&x, s, workspace, (hipStream_t)stream));
    HIP_TRY(launch_weights(w, a->dtype, (hipStream_t)stream));
    return SDPA_OK;
}

int sdpa_dev_evict_cache(const struct sdpa_heads *a, void *workspace, size_t workspace_bytes, void *stream) {
    (void)workspace; (void)workspace_bytes;
    SDPA_TRY(check_evict(a));
    if (a->batch == 0) return SDPA_OK;
    SDPA_TRY(require_device());
    EvictArgs x = {};
    x.k = a->k; x.v = a->v; x.k_out = a->k_out; x.v_out = a->v_out;
    x.w_in = a->weights; x.w_out = a->weights_out;
    x.wi_batch = a->weights_batch; x.wi_head = a->weights_head; x.wo_batch = a->weights_out_batch; x.wo_head = a->weights_out_head;
    x.lens = a->kv_lens; x.lens_out = a->lens_out; x.kept = a->kept;
    x.B = a->batch; x.Tk = a->kv_tokens; x.H = a->kv_heads; x.Dk = a->dk; x.Dv = a->dv;
    x.budget = a->budget; x.sinks = a->sinks; x.recent = a->recent;
    x.elem = elem_bytes(a->dtype);
    x.vec = rows_vec(a->k, a->dk, a->dtype) && rows_vec(a->k_out, a->dk, a->dtype) && rows_vec(a->v, a->dv, a->dtype) &&
            rows_vec(a->v_out, a->dv, a->dtype);
    HIP_TRY(launch_evict(x, (hipStream_t)stream));
    return SDPA_OK;
}

}  // extern "C"
