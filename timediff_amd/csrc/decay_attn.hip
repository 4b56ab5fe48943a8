// Decay attention (include/timediff_hip.h): S_t = g S_{t-1} + k_t v_t^T, o_t = scale S_t^T q_t, one decay g a head.
//
// One recurrence serves the operator and its gradients.  With rows a, b (da wide) and c (dc wide) and a state M (da x dc),
//     M_t = g M_{t-1} + us b_t c_t^T,      out_t = os M_t^T a_t
// is the forward pass for (a, b, c) = (q, k, v); the gradient of q for (grad_o, v, k) with the state transposed; and, run from
// the last row to the first, the gradient of v for (k, q, grad_o) and that of k for (v, grad_o, q), where M is the gradient of
// the state BEHIND a row: it enters a row undecayed and decays when it leaves it.
// The decay's gradient is sum_t <grad_o_t, d o_t / d log g>, and d M_t / d log g = g (M'_{t-1} + M_{t-1}) is carried beside M in the
// pass that computes grad_q: a sum without cancellation, where sum_t t (q.grad_q - k.grad_k) would lose everything for fast decays.
#include "decay_chunk.h"

using namespace decay;

namespace {

template <typename T> __device__ __forceinline__ float as_float(T x) { return (float)x; }

// The state entering each segment from what each segment adds: in place, one thread an element
template <bool TAN> __global__ __launch_bounds__(256) void td_decay_scan_kernel(Pass P) {
    const int size = P.da * P.dc, blocks = (size + 255) / 256, el = blockIdx.x % blocks * 256 + threadIdx.x;
    const int h = blockIdx.x / blocks % P.heads, n = blockIdx.x / blocks / P.heads;
    int lo, hi;
    row_range(P.offsets, P.rows, n, lo, hi);
    const int segments = (hi - lo + P.seg_len - 1) / P.seg_len;
    if (segments < 2 || el >= size) return;
    const double whole_d = exp((double)P.log_decay[h] * P.seg_len);
    const float whole = (float)whole_d;
    const int64_t first = P.offsets ? first_slot(P, n) : (int64_t)n * P.segs, by = (int64_t)P.heads * size;
    float *seg = P.seg + (first * P.heads + h) * size + el, *tan = TAN ? P.seg_tan + (first * P.heads + h) * size + el : nullptr;
    float F = P.state_in ? P.state_in[((int64_t)n * P.heads + h) * size + el] : 0.0f, H = 0.0f;
    float add = seg[0], add_tan = TAN ? tan[0] : 0.0f;
    for (int p = 1; p < segments; ++p) {
        const float next = p < segments - 1 ? seg[p * by] : 0.0f, next_tan = TAN && p < segments - 1 ? tan[p * by] : 0.0f;
        if (TAN) tan[p * by] = H = whole * (H + (float)P.seg_len * F) + add_tan;
        seg[p * by] = F = whole * F + add;
        add = next;
        add_tan = next_tan;
    }
}

// grad_log_decay[h] = the sum of head h's parts, in their order
__global__ __launch_bounds__(256) void td_decay_slope_kernel(const double *parts, int n, int heads, float *grad) {
    __shared__ double red[256];
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += 256) s += parts[(int64_t)i * heads + blockIdx.x];
    red[threadIdx.x] = s;
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1) {
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

// Rows of no sequence: zeros
template <typename T>
__global__ __launch_bounds__(256) void td_decay_clear_kernel(const int32_t *offsets, int n_seq, int rows, int width, T *out) {
    const int lo = min(max(offsets[0], 0), rows), hi = min(max(offsets[n_seq], lo), rows);
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x)
        if (row < lo || row >= hi)
            for (int i = threadIdx.x; i < width; i += 256) out[row * width + i] = (T)0.0f;
}

template <typename T>
__global__ __launch_bounds__(256) void td_decay_step_kernel(Pass P) {
    constexpr int D = TD_DECAY_MAX_DIM;
    __shared__ float part[256];
    const int h = blockIdx.x % P.heads, n = blockIdx.x / P.heads, tid = threadIdx.x, col = tid & (D - 1), half = tid / D;
    const float g = expf(P.log_decay[h]);
    float sum = 0.0f;
    if (col < P.dc) {
        const T *a = base_of<T>(P.a, false, n, h), *b = base_of<T>(P.b, false, n, h);
        const float c = as_float<T>(base_of<T>(P.c, false, n, h)[col]);
        float *S = P.state_out + (int64_t)blockIdx.x * P.da * P.dc + col;
        for (int i = half; i < P.da; i += 2) {
            const float s = g * S[(int64_t)i * P.dc] + as_float<T>(b[i]) * c;
            S[(int64_t)i * P.dc] = s;
            sum += as_float<T>(a[i]) * s;
        }
    }
    part[tid] = sum;
    __syncthreads();
    if (half == 0 && col < P.dc) ((T *)P.out)[(int64_t)blockIdx.x * P.dc + col] = (T)((part[tid] + part[tid + D]) * P.out_scale);
}

// ---- host side -----------------------------------------------------------------------------------------------------------
int check_config(const td_decay_config *c) {
    TD_REQUIRE(c, "configuration required");
    TD_REQUIRE(c->n_seq >= 1, "n_seq must be at least 1, got %d", c->n_seq);
    TD_REQUIRE(c->rows >= 0, "rows must not be negative, got %d", c->rows);
    TD_REQUIRE(c->packed == 0 || c->packed == 1, "packed must be 0 or 1, got %d", c->packed);
    TD_REQUIRE(c->dtype == TD_F32 || c->dtype == TD_BF16, "dtype must be TD_F32 or TD_BF16, got %d", c->dtype);
    TD_REQUIRE(c->dk >= 1 && c->dk <= TD_DECAY_MAX_DIM && c->dv >= 1 && c->dv <= TD_DECAY_MAX_DIM,
               "dk and dv must be 1 .. %d, got %d and %d", TD_DECAY_MAX_DIM, c->dk, c->dv);
    TD_REQUIRE(c->heads >= 1 && c->q_heads >= 1 && c->k_heads >= 1 && c->v_heads >= 1 && c->heads % c->q_heads == 0 &&
                   c->heads % c->k_heads == 0 && c->heads % c->v_heads == 0,
               "q_heads, k_heads and v_heads must divide heads, got %d, %d, %d and %d", c->q_heads, c->k_heads, c->v_heads, c->heads);
    TD_REQUIRE(((int64_t)c->n_seq + c->rows / CHUNK) * c->heads * ((c->dk * c->dv + 255) / 256) < (1LL << 31) &&
                   (int64_t)c->n_seq * (c->rows / 256 + 1) * c->heads < (1LL << 31),
               "too many sequences, rows and heads for one launch: n_seq %d, rows %d, heads %d", c->n_seq, c->rows, c->heads);
    TD_REQUIRE((int64_t)c->heads * TD_DECAY_MAX_DIM * CHUNK * 4 < (1LL << 31), "heads must be below 65536, got %d", c->heads);
    return TD_OK;
}

int64_t total_rows(const td_decay_config *c) { return c->packed ? c->rows : (int64_t)c->n_seq * c->rows; }
size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

int esize(const td_decay_config *c) { return c->dtype == TD_BF16 ? 2 : 4; }

View view(const td_decay_config *c, const void *p, const int64_t *s, int own, int d) { return View{p, s[0], s[1], s[2], c->heads / own, d}; }

// Whether a tensor can be read 16 bytes at a time, a chunk's rows at 32-bit offsets from its first
bool wide(const td_decay_config *c, const View &v) {
    const int64_t per = 16 / esize(c);
    return (uintptr_t)v.p % 16 == 0 && v.d % per == 0 && v.seq % per == 0 && v.row % per == 0 && v.head % per == 0 && v.row >= 0 &&
           v.row < (1LL << 31) / CHUNK / 4;
}

// Segments: enough workgroups to fill the chip (1024: four a compute unit), each of 256 rows at least
void split(const td_decay_config *c, int &len, int &segs, int64_t &slots) {
    const int64_t rows = total_rows(c), want = rows * c->heads / 1024;
    int64_t l = (want > 256 ? want : 256) + CHUNK - 1;
    l -= l % CHUNK;
    const int64_t longest = c->rows;
    if (l >= longest) {
        len = (int)(longest > 1 ? longest : 1);
        segs = 1;
        slots = c->n_seq;
    } else {
        len = (int)l;
        segs = c->packed ? 0 : (int)((longest + l - 1) / l);
        slots = c->packed ? c->rows / l + c->n_seq : (int64_t)c->n_seq * segs;
    }
}

Pass base_pass(const td_decay_config *c, const float *log_decay, const int32_t *offsets) {
    Pass P = {};
    P.log_decay = log_decay;
    P.offsets = c->packed ? offsets : nullptr;
    P.n_seq = c->n_seq;
    P.rows = c->rows;
    P.heads = c->heads;
    P.out_scale = P.upd_scale = 1.0f;
    int64_t slots;
    split(c, P.seg_len, P.segs, slots);
    P.slots = (int)slots;
    return P;
}

template <typename T, int DP, int NW, int CT, bool VEC, Form FORM, int WAVES> int launch(const Pass &P, hipStream_t st) {
    hipLaunchKernelGGL((td_decay_chunk_kernel<T, DP, NW, CT, VEC, FORM, WAVES>), dim3((unsigned)(P.slots * P.heads)), dim3(64 * NW), 0, st, P);
    TD_LAUNCH_CHECK();
    return TD_OK;
}

template <typename T, bool VEC, Form FORM> int launch_d(const Pass &P, hipStream_t st) {
    constexpr bool tan = FORM == OUT_TANGENT || FORM == SUM_TANGENT;
    const int d = P.da > P.dc ? P.da : P.dc;
    if (d <= 32) return launch<T, 32, 2, 1, VEC, FORM, 3>(P, st);
    if (d <= 64) return launch<T, 64, 4, 1, VEC, FORM, tan ? 2 : 3>(P, st);
    return launch<T, 128, 4, 2, VEC, FORM, tan ? 1 : 2>(P, st);
}

template <Form FORM> int launch_form(const td_decay_config *c, const Pass &P, hipStream_t st) {
    constexpr bool add = FORM == SUM || FORM == SUM_TANGENT;
    const bool vec = wide(c, P.b) && wide(c, P.c) && (add || (wide(c, P.a) && (uintptr_t)P.out % 16 == 0)) && (FORM != OUT_TANGENT || wide(c, P.e));
    if (c->dtype == TD_BF16) return vec ? launch_d<__bf16, true, FORM>(P, st) : launch_d<__bf16, false, FORM>(P, st);
    return vec ? launch_d<float, true, FORM>(P, st) : launch_d<float, false, FORM>(P, st);
}

// What the segments add, and the state that enters each of them (nothing to do where every sequence is one segment)
template <bool TAN> int enter_states(const td_decay_config *c, const Pass &P, hipStream_t st) {
    if (P.segs == 1) return TD_OK;
    if (int rc = launch_form<TAN ? SUM_TANGENT : SUM>(c, P, st)) return rc;
    const int64_t blocks = (int64_t)P.n_seq * P.heads * ((P.da * P.dc + 255) / 256);
    hipLaunchKernelGGL(td_decay_scan_kernel<TAN>, dim3((unsigned)blocks), dim3(256), 0, st, P);
    TD_LAUNCH_CHECK();
    return TD_OK;
}

int clear_rows(const td_decay_config *c, const int32_t *offsets, int width, void *out, hipStream_t st) {
    if (!c->packed || c->rows == 0) return TD_OK;
    const dim3 grid(c->rows < 256 ? c->rows : 256);
    if (c->dtype == TD_BF16) hipLaunchKernelGGL(td_decay_clear_kernel<__bf16>, grid, dim3(256), 0, st, offsets, c->n_seq, c->rows, width, (__bf16 *)out);
    else hipLaunchKernelGGL(td_decay_clear_kernel<float>, grid, dim3(256), 0, st, offsets, c->n_seq, c->rows, width, (float *)out);
    TD_LAUNCH_CHECK();
    return TD_OK;
}

// One gradient: straight into `grad` where every head has its own, else into float32 `parts` and their sum
int grad_pass(const td_decay_config *c, Pass P, int own_heads, int d, void *grad, float *parts, bool tangent, hipStream_t st) {
    const bool shared = own_heads != c->heads;
    P.out = !grad ? nullptr : shared ? (void *)parts : grad;
    P.out_f32 = shared;
    int rc = tangent ? launch_form<OUT_TANGENT>(c, P, st) : launch_form<OUT>(c, P, st);
    if (rc != TD_OK || !grad) return rc;
    const int64_t n = total_rows(c) * own_heads * d;
    if (shared && n > 0) {
        const int64_t blocks = (n + 255) / 256;
        const dim3 grid((unsigned)(blocks > 8192 ? 8192 : blocks));
        if (c->dtype == TD_BF16)
            hipLaunchKernelGGL(td_decay_share_sum_kernel<__bf16>, grid, dim3(256), 0, st, parts, (__bf16 *)grad, n, c->heads / own_heads, d);
        else
            hipLaunchKernelGGL(td_decay_share_sum_kernel<float>, grid, dim3(256), 0, st, parts, (float *)grad, n, c->heads / own_heads, d);
        TD_LAUNCH_CHECK();
    }
    return clear_rows(c, P.offsets, own_heads * d, grad, st);
}

struct Layout { size_t seg, seg_tan, slope, parts, total; };
Layout layout(const td_decay_config *c, bool backward) {
    int len, segs;
    int64_t slots;
    split(c, len, segs, slots);
    const size_t states = segs == 1 ? 0 : up256((size_t)slots * c->heads * c->dk * c->dv * sizeof(float));
    const bool shared = c->q_heads != c->heads || c->k_heads != c->heads || c->v_heads != c->heads;
    const int d = c->dk > c->dv ? c->dk : c->dv;
    Layout w;
    w.seg = 0;
    w.seg_tan = states;
    w.slope = w.seg_tan + (backward ? states : 0);
    w.parts = w.slope + (backward ? up256((size_t)slots * c->heads * sizeof(double)) : 0);
    w.total = w.parts + (backward && shared ? up256((size_t)total_rows(c) * c->heads * d * sizeof(float)) : 256);
    return w;
}

}  // namespace

extern "C" size_t td_decay_workspace_bytes(const td_decay_config *cfg, int32_t backward) {
    if (check_config(cfg) != TD_OK) return 0;
    return layout(cfg, backward != 0).total;
}

extern "C" int td_decay_forward(const td_decay_config *cfg, const void *q, const void *k, const void *v, const float *log_decay,
                                const int32_t *offsets, const float *state_in, void *o, float *state_out, void *workspace, void *stream) {
    if (int rc = check_config(cfg)) return rc;
    TD_REQUIRE(log_decay && workspace && (cfg->rows == 0 || (q && k && v && o)), "null pointer");
    TD_REQUIRE(!cfg->packed || offsets, "packed sequences need offsets");
    TD_REQUIRE(!state_out || state_out != state_in, "state_in and state_out must not be the same memory");
    Pass P = base_pass(cfg, log_decay, offsets);
    P.a = view(cfg, q, cfg->q_stride, cfg->q_heads, cfg->dk);
    P.b = view(cfg, k, cfg->k_stride, cfg->k_heads, cfg->dk);
    P.c = view(cfg, v, cfg->v_stride, cfg->v_heads, cfg->dv);
    P.da = cfg->dk; P.dc = cfg->dv; P.st_a = cfg->dv; P.st_c = 1;
    P.state_in = state_in; P.state_out = state_out;
    P.out = o; P.out_scale = cfg->scale;
    P.seg = (float *)workspace;
    if (int rc = enter_states<false>(cfg, P, (hipStream_t)stream)) return rc;
    if (int rc = launch_form<OUT>(cfg, P, (hipStream_t)stream)) return rc;
    return clear_rows(cfg, offsets, cfg->heads * cfg->dv, o, (hipStream_t)stream);
}

extern "C" int td_decay_backward(const td_decay_config *cfg, const void *q, const void *k, const void *v, const float *log_decay,
                                 const int32_t *offsets, const float *state_in, const void *grad_o, const float *grad_state_out, void *grad_q,
                                 void *grad_k, void *grad_v, float *grad_log_decay, float *grad_state_in, void *workspace, void *stream) {
    if (int rc = check_config(cfg)) return rc;
    TD_REQUIRE(log_decay && workspace && (cfg->rows == 0 || (q && k && v && grad_o)), "null pointer");
    TD_REQUIRE(!cfg->packed || offsets, "packed sequences need offsets");
    hipStream_t st = (hipStream_t)stream;
    const Layout w = layout(cfg, true);
    float *parts = (float *)((char *)workspace + w.parts);
    const View vq = view(cfg, q, cfg->q_stride, cfg->q_heads, cfg->dk), vk = view(cfg, k, cfg->k_stride, cfg->k_heads, cfg->dk),
               vv = view(cfg, v, cfg->v_stride, cfg->v_heads, cfg->dv), vo = view(cfg, grad_o, cfg->grad_o_stride, cfg->heads, cfg->dv);
    if (grad_q || grad_log_decay) {
        Pass P = base_pass(cfg, log_decay, offsets);
        P.a = vo; P.b = vv; P.c = vk; P.e = vq;
        P.da = cfg->dv; P.dc = cfg->dk; P.st_a = 1; P.st_c = cfg->dv;
        P.state_in = state_in; P.grad_state = grad_state_out; P.slope = (double *)((char *)workspace + w.slope);
        P.out_scale = cfg->scale;
        P.seg = (float *)((char *)workspace + w.seg); P.seg_tan = (float *)((char *)workspace + w.seg_tan);
        if (int rc = grad_log_decay ? enter_states<true>(cfg, P, st) : enter_states<false>(cfg, P, st)) return rc;
        if (int rc = grad_pass(cfg, P, cfg->q_heads, cfg->dk, grad_q, parts, grad_log_decay != nullptr, st)) return rc;
        if (grad_log_decay) {
            hipLaunchKernelGGL(td_decay_slope_kernel, dim3(cfg->heads), dim3(256), 0, st, P.slope, P.slots, cfg->heads, grad_log_decay);
            TD_LAUNCH_CHECK();
        }
    }
    if (grad_v || grad_k || grad_state_in) {
        Pass P = base_pass(cfg, log_decay, offsets);
        P.reverse = 1;
        P.a = vk; P.b = vq; P.c = vo;
        P.da = cfg->dk; P.dc = cfg->dv; P.st_a = cfg->dv; P.st_c = 1;
        P.state_in = grad_state_out; P.upd_scale = cfg->scale;
        P.seg = (float *)((char *)workspace + w.seg);
        if (int rc = enter_states<false>(cfg, P, st)) return rc;
        if (grad_v || grad_state_in) {
            P.state_out = grad_state_in;
            if (int rc = grad_pass(cfg, P, cfg->v_heads, cfg->dv, grad_v, parts, false, st)) return rc;
        }
        if (grad_k) {
            P.state_out = nullptr;
            P.a = vv; P.b = vo; P.c = vq;
            P.da = cfg->dv; P.dc = cfg->dk; P.st_a = 1; P.st_c = cfg->dv;
            if (int rc = grad_pass(cfg, P, cfg->k_heads, cfg->dk, grad_k, parts, false, st)) return rc;
        }
    }
    return TD_OK;
}

extern "C" int td_decay_step(const td_decay_config *cfg, const void *q, const void *k, const void *v, const float *log_decay, float *state,
                             void *o, void *stream) {
    if (int rc = check_config(cfg)) return rc;
    TD_REQUIRE(cfg->rows == 1 && !cfg->packed, "td_decay_step takes one row of each sequence (rows = 1, packed = 0)");
    TD_REQUIRE(q && k && v && log_decay && state && o, "null pointer");
    Pass P = base_pass(cfg, log_decay, nullptr);
    P.a = view(cfg, q, cfg->q_stride, cfg->q_heads, cfg->dk);
    P.b = view(cfg, k, cfg->k_stride, cfg->k_heads, cfg->dk);
    P.c = view(cfg, v, cfg->v_stride, cfg->v_heads, cfg->dv);
    P.da = cfg->dk; P.dc = cfg->dv;
    P.state_out = state; P.out = o; P.out_scale = cfg->scale;
    const dim3 grid(cfg->n_seq * cfg->heads);
    if (cfg->dtype == TD_BF16) hipLaunchKernelGGL(td_decay_step_kernel<__bf16>, grid, dim3(256), 0, (hipStream_t)stream, P);
    else hipLaunchKernelGGL(td_decay_step_kernel<float>, grid, dim3(256), 0, (hipStream_t)stream, P);
    TD_LAUNCH_CHECK();
    return TD_OK;
}
