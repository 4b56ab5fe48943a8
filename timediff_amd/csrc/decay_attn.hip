// Decay attention (include/timediff_hip.h): S_t = g S_{t-1} + k_t v_t^T, o_t = scale S_t^T q_t, one decay g a head.
//
// One recurrence serves the operator and its gradients.  With rows a, b (da wide) and c (dc wide) and a state M (da x dc),
//     M_t = g M_{t-1} + us b_t c_t^T,      out_t = os M_t^T a_t
// is the forward pass for (a, b, c) = (q, k, v); the gradient of q for (grad_o, v, k) with the state transposed; and, run from
// the last row to the first, the gradient of v for (k, q, grad_o) and that of k for (v, grad_o, q), where M is the gradient of
// the state BEHIND a row: it enters a row undecayed and decays when it leaves it.
//
// The gradient by log g is sum over t >= s of (t - s) g^(t-s) (q_t . k_s)(v_s . grad_o_t) and the entering state's like terms.  The number
// of rows from s to t is cut where chunks begin: rows of t's chunk up to t (from grad_q's part that the state entering that chunk made, row
// by row), rows of s's chunk behind s (from grad_k's part that the chunks behind it made), and the n rows of every chunk between (n times
// the product of the state entering it and the gradient of the state leaving it).  Nothing cancels, where the shorter
// sum_t t (q_t . grad_q_t - k_t . grad_k_t) would lose everything for decays that forget within a few rows.
#include "decay_chunk.h"

using namespace decay;

// decay_inst.hip: one launcher per (element type, kernel)
#define TD_LAUNCHERS(b)                                                                                                              \
    int td_decay_launch_##b##_0(const Work &, int, hipStream_t); int td_decay_launch_##b##_1(const Work &, int, hipStream_t);       \
    int td_decay_launch_##b##_2(const Work &, int, hipStream_t); int td_decay_launch_##b##_3(const Work &, int, hipStream_t);       \
    int td_decay_launch_##b##_4(const Work &, int, hipStream_t);
TD_LAUNCHERS(0)
TD_LAUNCHERS(1)

namespace {

template <typename T> __device__ __forceinline__ float as_float(T x) { return (float)x; }

// The state entering each segment (REV: its gradient behind each segment) from what each segment adds: in place, one thread an element
template <bool REV> __global__ __launch_bounds__(256) void td_decay_scan_kernel(Pass P) {
    const int size = P.da * P.dc, blocks = (size + 255) / 256, place = P.first + blockIdx.x, el = place % blocks * 256 + threadIdx.x;
    const int h = place / blocks % P.heads, n = place / blocks / P.heads;
    int lo, hi;
    row_range(P.offsets, P.rows, n, lo, hi);
    const int segments = hi > lo ? (hi - lo - 1) / P.seg_len + 1 : 0;
    if (segments < 2 || el >= size) return;
    const float ld = P.log_decay[h];
    const Factor whole = factor(ld, P.seg_len);
    const int64_t first = P.offsets ? first_place(P, n, P.seg_len) : (int64_t)n * P.segs, by = (int64_t)P.heads * size;
    float *seg = P.seg + (first * P.heads + h) * size + el;
    float F = P.state_in ? P.state_in[((int64_t)n * P.heads + h) * size + el] : 0.0f;
    if (REV) {
        seg += (segments - 1) * by;
        float add = seg[0];
        seg[0] = F;
        F = times(factor(ld, hi - lo - (segments - 1) * P.seg_len), F) + add;
    } else {
        F = times(whole, F) + seg[0];
    }
    constexpr int AHEAD = 8;          // the loads do not wait for the sums
    for (int p = 1; p < segments; p += AHEAD) {
        float add[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) add[k] = p + k < segments - 1 ? seg[(REV ? -(p + k) : p + k) * by] : 0.0f;
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
            if (p + k < segments) {
                seg[(REV ? -(p + k) : p + k) * by] = F;
                F = times(whole, F) + add[k];
            }
    }
}

// grad_log_decay[h] = the sum of head h's parts, in an order of their own
__global__ __launch_bounds__(1024) void td_decay_slope_kernel(const double *parts, int64_t n, int heads, float *grad) {
    __shared__ double red[1024];
    double s = 0.0;
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < n; i += 1024) s += parts[i * heads + blockIdx.x];
    red[threadIdx.x] = s;
    __syncthreads();
    for (int o = 512; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) grad[blockIdx.x] = (float)red[0];
}

// The gradient of a tensor with fewer heads: the sum over the heads that share one of its own, rounded once
template <typename T>
__global__ __launch_bounds__(256) void td_decay_share_sum_kernel(const float *__restrict__ parts, T *__restrict__ out, int64_t n, int share, int d) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t head = i / d;
        const float *p = parts + head * share * d + (i - head * d);
        float s = 0.0f;
        for (int j = 0; j < share; ++j) s += p[(int64_t)j * d];
        out[i] = (T)s;
    }
}

// One row: a workgroup of NT threads for each state, W threads across its columns, the NT / W groups of them sharing out the rows.  Bound by memory:
// the state is read and written once (1024 x 8 states of 128 x 128: 4.4 TB/s).  W: the least of 16, 32, 64 and 128 that has every column (with
// 128 for all of them 2048 x 8 states of 64 x 64 take 167 us, with 64 126; 4096 x 8 of 32 x 32 float32 112 and 55).
template <typename T, int W, int NT>
__global__ __launch_bounds__(NT) void td_decay_step_kernel(Pass P) {
    constexpr int GROUPS = NT / W;
    __shared__ float part[NT];
    const int item = P.first + blockIdx.x, h = item % P.heads, n = item / P.heads, tid = threadIdx.x, col = tid % W, group = tid / W;
    const float g = expf(P.log_decay[h]);
    float sum = 0.0f;
    if (col < P.dc) {
        const T *a = base_of<T>(P.a, false, n, h), *b = base_of<T>(P.b, false, n, h);
        const float c = as_float<T>(base_of<T>(P.c, false, n, h)[col]);
        float *S = P.state_out + (int64_t)item * P.da * P.dc + col;
#pragma unroll 4
        for (int i = group; i < P.da; i += GROUPS) {
            const float s = g * S[(int64_t)i * P.dc] + as_float<T>(b[i]) * c;
            S[(int64_t)i * P.dc] = s;
            sum += as_float<T>(a[i]) * s;
        }
    }
    part[tid] = sum;
    __syncthreads();
    if (group == 0 && col < P.dc) {
#pragma unroll
        for (int k = 1; k < GROUPS; ++k) sum += part[tid + k * W];
        ((T *)P.out)[(int64_t)item * P.dc + col] = (T)(sum * P.out_scale);
    }
}
template <typename T, int NT> void launch_step(const Pass &P, hipStream_t st) {
    launch_parts(P, (int64_t)P.n_seq * P.heads, NT, [&](const Pass &P, dim3 grid) {
        const dim3 block(NT);
        if (NT == 256 && P.dc <= 16) hipLaunchKernelGGL((td_decay_step_kernel<T, 16, 256>), grid, block, 0, st, P);
        else if (P.dc <= 32) hipLaunchKernelGGL((td_decay_step_kernel<T, 32, NT>), grid, block, 0, st, P);
        else if (P.dc <= 64) hipLaunchKernelGGL((td_decay_step_kernel<T, 64, NT>), grid, block, 0, st, P);
        else hipLaunchKernelGGL((td_decay_step_kernel<T, 128, NT>), grid, block, 0, st, P);
    });
}
// Few states that are not small: 1024 threads for each, of which the chip holds 512 (64 x 8 states of 128 x 128: 14 us a call, 19 with 256 threads; 65 x 8
// take 22, with 256)
template <typename T> void launch_step(const Pass &P, hipStream_t st) {
    if (P.n_seq * P.heads <= 512 && P.da * P.dc >= 4096) launch_step<T, 1024>(P, st);
    else launch_step<T, 256>(P, st);
}

// ---- host side -----------------------------------------------------------------------------------------------------------
int check_config(const td_decay_config *c) {
    TD_REQUIRE(c, "configuration required");
    TD_REQUIRE(c->n_seq >= 1, "n_seq must be at least 1, got %d", c->n_seq);
    // (a chunk's first row and the one behind it are counted in 32 bits)
    TD_REQUIRE(c->rows >= 0 && c->rows <= INT32_MAX - 2 * CHUNK, "rows must be 0 .. %d, got %d", INT32_MAX - 2 * CHUNK, c->rows);
    TD_REQUIRE(c->packed == 0 || c->packed == 1, "packed must be 0 or 1, got %d", c->packed);
    TD_REQUIRE(c->dtype == TD_F32 || c->dtype == TD_BF16, "dtype must be TD_F32 or TD_BF16, got %d", c->dtype);
    TD_REQUIRE(c->dk >= 1 && c->dk <= TD_DECAY_MAX_DIM && c->dv >= 1 && c->dv <= TD_DECAY_MAX_DIM,
               "dk and dv must be 1 .. %d, got %d and %d", TD_DECAY_MAX_DIM, c->dk, c->dv);
    TD_REQUIRE(c->heads >= 1 && c->q_heads >= 1 && c->k_heads >= 1 && c->v_heads >= 1 && c->heads % c->q_heads == 0 &&
                   c->heads % c->k_heads == 0 && c->heads % c->v_heads == 0,
               "q_heads, k_heads and v_heads must divide heads, got %d, %d, %d and %d", c->q_heads, c->k_heads, c->v_heads, c->heads);
    TD_REQUIRE(((int64_t)c->n_seq + c->rows / CHUNK) * c->heads * ((c->dk * c->dv + 255) / 256) < (1LL << 31) &&
                   (int64_t)c->n_seq * (c->rows / 256 + 1) * c->heads < (1LL << 31),
               "too many sequences, rows and heads for one call: n_seq %d, rows %d, heads %d", c->n_seq, c->rows, c->heads);
    TD_REQUIRE((int64_t)c->heads * TD_DECAY_MAX_DIM * CHUNK * 4 < (1LL << 31), "heads must be below 65536, got %d", c->heads);
    return TD_OK;
}

int64_t total_rows(const td_decay_config *c) { return c->packed ? c->rows : (int64_t)c->n_seq * c->rows; }
size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

int esize(const td_decay_config *c) { return c->dtype == TD_BF16 ? 2 : 4; }

View view(const td_decay_config *c, const void *p, const int64_t *s, int own, int d) {
    const bool even = (uintptr_t)p % 4 == 0 && d % 2 == 0 && s[0] % 2 == 0 && s[1] % 2 == 0 && s[2] % 2 == 0;
    return View{p, s[0], s[1], s[2], c->heads / own, d, even};
}

// Whether a tensor can be read 16 bytes at a time, a chunk's rows at 32-bit offsets from its first (24 bits of row stride)
bool wide(const td_decay_config *c, const View &v) {
    const int64_t per = 16 / esize(c);
    return (uintptr_t)v.p % 16 == 0 && v.d % per == 0 && v.seq % per == 0 && v.row % per == 0 && v.head % per == 0 && v.row >= 0 &&
           v.row * esize(c) < (1 << 24);
}

// Segments: a sequence on its own is one after another, chunk by chunk, so few long ones are cut until the chip is full, which costs two launches
// and a second reading of k and v.  Measured (bfloat16, forward / backward):
//   * rows of a segment: 256 at least: the chip is full with 512 workgroups (two a compute unit), or with 256 where one workgroup's registers fill
//     a compute unit (backward of wide states): cut for 256 instead of 512 those backward passes take 371 instead of 409 us at 128
//     sequences and heads of 1024 rows, 128 x 128;
//   * nothing is cut up to 512 rows: 1, 4 and 8 sequences of 512 rows, 8 heads, 64 x 64, take 25, 26 and 26 us whole and 27, 29 and 30 cut in two
//     forward (128 x 128: 47, 48 and 48; 46, 51 and 55).  Backward they would gain: 87, 88 and 88 whole, 77, 79 and 83 cut (128 x 128: 164, 173
//     and 177; 138, 152 and 166);
//   * with a workgroup for three in four compute units nothing is cut: 256 of 1024 rows, 128 x 128, take 103 us whole forward and 155 cut for 512.
//     States of 32 x 32 have less to do between their loads and gain up to 512: 256 of 2048 rows 84 / 233 us cut, 95 / 282
//     whole.  Lengths of packed sequences are not known here: one of them may be nearly all rows;
//   * the backward pass of log_decay keeps the states entering a segment's chunks (64 KB a chunk of 128 x 128), so its segments are 4096
//     rows at most: 2 GiB in 512 workgroups (4 in 1024), where a sequence of 32768 rows in one piece would take 16.
void split(const td_decay_config *c, bool backward, int &len, int &segs, int64_t &slots) {
    const int64_t rows = total_rows(c), longest = c->rows;
    const int most = c->dk > c->dv ? c->dk : c->dv;
    const bool one = backward && most > (c->dtype == TD_BF16 ? 64 : 32);
    int64_t l = rows * c->heads / (one ? 256 : 512);
    if (l < 256) l = 256;
    if (!c->packed && most > 32 && (int64_t)c->n_seq * c->heads >= 192 && l < longest) l = longest;
    if (backward && longest > 4096) {
        const int64_t pieces = (longest + 4095) / 4096, even = (longest + pieces - 1) / pieces;
        if (l > even) l = even;
    }
    l += CHUNK - 1;
    l -= l % CHUNK;
    if (l >= longest || longest <= 512) {
        len = (int)(longest > 1 ? longest : 1);
        segs = 1;
        slots = c->n_seq;
    } else {
        len = (int)l;
        segs = c->packed ? 0 : (int)((longest + l - 1) / l);
        slots = c->packed ? c->rows / l + c->n_seq : (int64_t)c->n_seq * segs;
    }
}

Pass base_pass(const td_decay_config *c, bool backward, const float *log_decay, const int32_t *offsets) {
    Pass P = {};
    P.log_decay = log_decay;
    P.offsets = c->packed ? offsets : nullptr;
    P.n_seq = c->n_seq;
    P.rows = c->rows;
    P.heads = c->heads;
    P.out_scale = P.upd_scale = 1.0f;
    int64_t slots;
    split(c, backward, P.seg_len, P.segs, slots);
    P.slots = (int)slots;
    return P;
}

int launch(const td_decay_config *c, Kind kind, const Work &w, bool vec, hipStream_t st) {
    typedef int (*Launcher)(const Work &, int, hipStream_t);
    static const Launcher table[2][5] = {
        {td_decay_launch_0_0, td_decay_launch_0_1, td_decay_launch_0_2, td_decay_launch_0_3, td_decay_launch_0_4},
        {td_decay_launch_1_0, td_decay_launch_1_1, td_decay_launch_1_2, td_decay_launch_1_3, td_decay_launch_1_4}};
    return table[c->dtype == TD_BF16][kind](w, vec, st);
}
int launch(const td_decay_config *c, Kind kind, const Pass &P, bool vec, hipStream_t st) {
    Work w = {};
    w.p = P;
    return launch(c, kind, w, vec, st);
}

// Workgroups of the backward pass, each with its own place for the states of a segment's chunks, one (slot, head) after another: as many as the
// chip holds, two a compute unit and, of bfloat16 states up to 32 x 32 (53 KB of LDS, two waves), three: 512 sequences of 272 rows, 8 heads,
// bfloat16: 319 us with 768 workgroups, 466 with 512, 440 with 1024; float32 (57 KB): 636, 517, 519 (before its states summed 32 rows first: with
// 512 524 now).  Packed slots have different lengths, and workgroups that wait for a place on the chip even that out (20011 rows of 40
// sequences, 8 heads of 64 x 128: 336 us with 512, 326 with 1024).
int backward_groups(const td_decay_config *c, int64_t slots) {
    const int64_t most = c->packed ? 1024 : c->dtype == TD_BF16 && c->dk <= 32 && c->dv <= 32 ? 768 : 512;
    return (int)(slots * c->heads < most ? slots * c->heads : most);
}

// What the segments add, and the state that enters each of them (nothing to do where every sequence is one segment)
template <bool REV> int enter_states(const td_decay_config *c, const Pass &P, bool vec, hipStream_t st) {
    if (P.segs == 1) return TD_OK;
    if (int rc = launch(c, REV ? SUM_REVERSED : SUM, P, vec, st)) return rc;
    const int64_t blocks = (int64_t)P.n_seq * P.heads * ((P.da * P.dc + 255) / 256);
    launch_parts(P, blocks, 256, [&](const Pass &P, dim3 grid) { hipLaunchKernelGGL(td_decay_scan_kernel<REV>, grid, dim3(256), 0, st, P); });
    TD_LAUNCH_CHECK();
    return TD_OK;
}

// The gradient of a tensor whose heads are shared, from float32 parts of every head
int share_sum(const td_decay_config *c, const float *parts, void *grad, int own_heads, int d, hipStream_t st) {
    const int64_t n = total_rows(c) * own_heads * d, blocks = (n + 255) / 256;
    if (n == 0) return TD_OK;
    const dim3 grid((unsigned)(blocks > 8192 ? 8192 : blocks));
    if (c->dtype == TD_BF16)
        hipLaunchKernelGGL(td_decay_share_sum_kernel<__bf16>, grid, dim3(256), 0, st, parts, (__bf16 *)grad, n, c->heads / own_heads, d);
    else
        hipLaunchKernelGGL(td_decay_share_sum_kernel<float>, grid, dim3(256), 0, st, parts, (float *)grad, n, c->heads / own_heads, d);
    TD_LAUNCH_CHECK();
    return TD_OK;
}

// Floats of the states of a segment's chunks in the backward kernel that decay_inst.hip takes
int64_t held_states(const td_decay_config *c, int len) {
    const int most = c->dk > c->dv ? c->dk : c->dv, side = most <= 32 ? 32 : 64;
    return (int64_t)(c->dk <= 64 ? side : 128) * (c->dv <= 64 ? side : 128) * ((len + CHUNK - 1) / CHUNK);
}

constexpr size_t NO_WORKSPACE = 256;      // what a call that uses none asks for: 0 says that the configuration is bad
struct Layout { size_t seg, seg2, chunks, slope, parts, parts2, parts3, total; };
// want: the `backward` of td_decay_workspace_bytes
Layout layout(const td_decay_config *c, int want) {
    const bool backward = want != 0, all = want == TD_DECAY_GRAD_ALL, slope = backward && (all || want & TD_DECAY_GRAD_LOG_DECAY);
    int len, segs;
    int64_t slots;
    split(c, backward, len, segs, slots);
    const size_t state = (size_t)c->heads * c->dk * c->dv * sizeof(float), rows = (size_t)total_rows(c) * c->heads * sizeof(float);
    Layout w;
    w.seg = 0;
    w.seg2 = segs == 1 ? 0 : up256(slots * state);
    w.chunks = w.seg2 + (backward && segs != 1 ? up256(slots * state) : 0);
    w.slope = w.chunks + (slope ? held_states(c, len) * sizeof(float) * backward_groups(c, slots) : 0);
    w.parts = w.slope + (slope ? up256(2 * (size_t)slots * c->heads * sizeof(double)) : 0);
    const auto part = [&](int bit, int own, int d) { return backward && (all || want & bit) && own != c->heads ? up256(rows * d) : 0; };
    w.parts2 = w.parts + part(TD_DECAY_GRAD_Q, c->q_heads, c->dk);
    w.parts3 = w.parts2 + part(TD_DECAY_GRAD_K, c->k_heads, c->dk);
    w.total = w.parts3 + part(TD_DECAY_GRAD_V, c->v_heads, c->dv) + NO_WORKSPACE;
    return w;
}

bool aligned(const void *p) { return (uintptr_t)p % 16 == 0; }

}  // namespace

extern "C" size_t td_decay_workspace_bytes(const td_decay_config *cfg, int32_t backward) {
    if (check_config(cfg) != TD_OK) return 0;
    constexpr int known = TD_DECAY_GRAD_ALL | TD_DECAY_GRAD_SOME | TD_DECAY_GRAD_Q | TD_DECAY_GRAD_K | TD_DECAY_GRAD_V | TD_DECAY_GRAD_LOG_DECAY;
    if (backward & ~known || (backward & ~TD_DECAY_GRAD_ALL && (backward & TD_DECAY_GRAD_ALL || !(backward & TD_DECAY_GRAD_SOME)))) {
        td_set_error("backward must be 0, TD_DECAY_GRAD_ALL or TD_DECAY_GRAD_SOME with others, got %d", backward);
        return 0;
    }
    return layout(cfg, backward).total;
}

extern "C" int td_decay_forward(const td_decay_config *cfg, const void *q, const void *k, const void *v, const float *log_decay,
                                const int32_t *offsets, const float *state_in, void *o, float *state_out, void *workspace, void *stream) {
    if (int rc = check_config(cfg)) return rc;
    TD_REQUIRE(log_decay && (workspace || layout(cfg, 0).total == NO_WORKSPACE) && (cfg->rows == 0 || (q && k && v && o)), "null pointer");
    TD_REQUIRE(!cfg->packed || offsets, "packed sequences need offsets");
    TD_REQUIRE(!state_out || state_out != state_in, "state_in and state_out must not be the same memory");
    hipStream_t st = (hipStream_t)stream;
    Pass P = base_pass(cfg, false, log_decay, offsets);
    P.a = view(cfg, q, cfg->q_stride, cfg->q_heads, cfg->dk);
    P.b = view(cfg, k, cfg->k_stride, cfg->k_heads, cfg->dk);
    P.c = view(cfg, v, cfg->v_stride, cfg->v_heads, cfg->dv);
    P.da = cfg->dk; P.dc = cfg->dv; P.st_a = cfg->dv; P.st_c = 1;
    P.state_in = state_in; P.state_out = state_out;
    P.out = o; P.out_scale = cfg->scale;
    P.seg = (float *)workspace;
    const bool vec = wide(cfg, P.a) && wide(cfg, P.b) && wide(cfg, P.c) && aligned(o);
    if (int rc = enter_states<false>(cfg, P, vec, st)) return rc;
    return launch(cfg, OUT, P, vec, st);
}

extern "C" int td_decay_backward(const td_decay_config *cfg, const void *q, const void *k, const void *v, const float *log_decay,
                                 const int32_t *offsets, const float *state_in, const void *grad_o, const float *grad_state_out, void *grad_q,
                                 void *grad_k, void *grad_v, float *grad_log_decay, float *grad_state_in, void *workspace, void *stream) {
    if (int rc = check_config(cfg)) return rc;
    const bool slope = grad_log_decay != nullptr;
    const Layout l = layout(cfg, TD_DECAY_GRAD_SOME | (grad_q ? TD_DECAY_GRAD_Q : 0) | (grad_k ? TD_DECAY_GRAD_K : 0) | (grad_v ? TD_DECAY_GRAD_V : 0) |
                                     (slope ? TD_DECAY_GRAD_LOG_DECAY : 0));
    TD_REQUIRE(log_decay && (workspace || l.total == NO_WORKSPACE) && (cfg->rows == 0 || (q && k && v && grad_o)), "null pointer");
    TD_REQUIRE(!cfg->packed || offsets, "packed sequences need offsets");
    hipStream_t st = (hipStream_t)stream;
    char *ws = (char *)workspace;
    const bool q_shared = cfg->q_heads != cfg->heads, k_shared = cfg->k_heads != cfg->heads, v_shared = cfg->v_heads != cfg->heads;
    float *parts_q = (float *)(ws + l.parts), *parts_k = (float *)(ws + l.parts2), *parts_v = (float *)(ws + l.parts3);
    const View vq = view(cfg, q, cfg->q_stride, cfg->q_heads, cfg->dk), vk = view(cfg, k, cfg->k_stride, cfg->k_heads, cfg->dk),
               vv = view(cfg, v, cfg->v_stride, cfg->v_heads, cfg->dv), vo = view(cfg, grad_o, cfg->grad_o_stride, cfg->heads, cfg->dv);
    const bool vec = wide(cfg, vq) && wide(cfg, vk) && wide(cfg, vv) && wide(cfg, vo) && aligned(grad_q) && aligned(grad_k) && aligned(grad_v);
    Work w = {};
    w.chunk_states = (float *)(ws + l.chunks);
    w.ascending = grad_q || slope;
    w.descending = grad_v || grad_k || grad_state_in || slope;
    Pass &Q = w.p, &R = w.r;
    Q = R = base_pass(cfg, true, log_decay, offsets);
    w.groups = backward_groups(cfg, Q.slots);
    double *slopes = (double *)(ws + l.slope);
    Q.a = vo; Q.b = vv; Q.c = vk; Q.e = vq;
    Q.da = cfg->dv; Q.dc = cfg->dk; Q.st_a = 1; Q.st_c = cfg->dv;
    Q.state_in = state_in; Q.slope = slopes; Q.out_scale = cfg->scale;
    Q.out = !grad_q ? nullptr : q_shared ? (void *)parts_q : grad_q;
    Q.out_f32 = q_shared;
    Q.seg = (float *)(ws + l.seg);
    R.a = vk; R.b = vq; R.c = vo; R.e = vv;
    R.da = cfg->dk; R.dc = cfg->dv; R.st_a = cfg->dv; R.st_c = 1;
    R.state_in = grad_state_out; R.state_out = grad_state_in; R.upd_scale = cfg->scale;
    R.slope = slopes + (size_t)R.slots * cfg->heads;
    R.out = !grad_v ? nullptr : v_shared ? (void *)parts_v : grad_v;
    R.out_f32 = v_shared;
    R.out2 = !grad_k ? nullptr : k_shared ? (void *)parts_k : grad_k;
    R.out2_f32 = k_shared;
    R.seg = (float *)(ws + l.seg2);
    if (w.ascending)
        if (int rc = enter_states<false>(cfg, Q, vec, st)) return rc;
    if (w.descending)
        if (int rc = enter_states<true>(cfg, R, vec, st)) return rc;
    if (w.ascending || w.descending)
        if (int rc = launch(cfg, slope ? BACKWARD_SLOPE : BACKWARD, w, vec, st)) return rc;
    if (grad_q && q_shared)
        if (int rc = share_sum(cfg, parts_q, grad_q, cfg->q_heads, cfg->dk, st)) return rc;
    if (grad_v && v_shared)
        if (int rc = share_sum(cfg, parts_v, grad_v, cfg->v_heads, cfg->dv, st)) return rc;
    if (grad_k && k_shared)
        if (int rc = share_sum(cfg, parts_k, grad_k, cfg->k_heads, cfg->dk, st)) return rc;
    if (slope) {
        hipLaunchKernelGGL(td_decay_slope_kernel, dim3(cfg->heads), dim3(1024), 0, st, slopes, 2 * (int64_t)Q.slots, cfg->heads, grad_log_decay);
        TD_LAUNCH_CHECK();
    }
    return TD_OK;
}

extern "C" int td_decay_step(const td_decay_config *cfg, const void *q, const void *k, const void *v, const float *log_decay, float *state,
                             void *o, void *stream) {
    if (int rc = check_config(cfg)) return rc;
    TD_REQUIRE(cfg->rows == 1 && !cfg->packed, "td_decay_step takes one row of each sequence (rows = 1, packed = 0)");
    TD_REQUIRE(q && k && v && log_decay && state && o, "null pointer");
    Pass P = base_pass(cfg, false, log_decay, nullptr);
    P.a = view(cfg, q, cfg->q_stride, cfg->q_heads, cfg->dk);
    P.b = view(cfg, k, cfg->k_stride, cfg->k_heads, cfg->dk);
    P.c = view(cfg, v, cfg->v_stride, cfg->v_heads, cfg->dv);
    P.da = cfg->dk; P.dc = cfg->dv;
    P.state_out = state; P.out = o; P.out_scale = cfg->scale;
    if (cfg->dtype == TD_BF16) launch_step<__bf16>(P, (hipStream_t)stream);
    else launch_step<float>(P, (hipStream_t)stream);
    TD_LAUNCH_CHECK();
    return TD_OK;
}
