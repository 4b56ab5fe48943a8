// Decay attention (include/timediff_hip.h): S_t = g S_{t-1} + k_t v_t^T, o_t = scale S_t^T q_t, one decay g a head.
//
// One recurrence serves the operator and its gradients.  With rows a, b (da wide) and c (dc wide) and a state M (da x dc),
//     M_t = g M_{t-1} + us b_t c_t^T,      out_t = os M_t^T a_t
// is the forward pass for (a, b, c) = (q, k, v); the gradient of q for (grad_o, v, k) with the state transposed; and, run from
// the last row to the first, the gradient of v for (k, q, grad_o) and that of k for (v, grad_o, q), where M is the gradient of
// the state BEHIND a row: it enters a row undecayed and decays when it leaves it.
// The decay's gradient is sum_t <grad_o_t, d o_t / d log g>, and d M_t / d log g = g (M'_{t-1} + M_{t-1}) is carried beside M in the
// pass that computes grad_q: a sum without cancellation, where sum_t t (q.grad_q - k.grad_k) would lose everything for fast decays.
#include "common.h"

namespace {

struct View {                 // rows of one tensor; head h of the recurrence reads head h / share
    const void *p;
    int64_t seq, row, head;
    int share;
};

struct Pass {
    View a, b, c, e;          // e: what the tangent's output is dotted with (tangent form only)
    const float *log_decay;
    const int32_t *offsets;   // packed: n_seq + 1, else NULL
    const float *state_in;    // (n_seq, heads, ..): element (i, j) of (da, dc) at i * st_a + j * st_c, NULL: zeros
    float *state_out;         // NULL: not wanted
    const float *grad_state;  // tangent form: the gradient of the state left behind, NULL: none
    double *slope;            // tangent form: one sum for each (sequence, head)
    int64_t st_a, st_c;
    void *out;                // (rows, heads, dc), float32 (out_f32) or the tensors' type; NULL: not wanted
    int out_f32;
    int n_seq, rows, heads, da, dc, reverse;
    float out_scale, upd_scale;
};

template <typename T> __device__ __forceinline__ float as_float(T x);
template <> __device__ __forceinline__ float as_float<float>(float x) { return x; }
template <> __device__ __forceinline__ float as_float<__bf16>(__bf16 x) { return (float)x; }

// g^e for a whole number e: 1 for e = 0, also where log g is -inf
__device__ __forceinline__ float decay_pow(float lg2, int e) { return e == 0 ? 1.0f : exp2f(lg2 * (float)e); }

// The rows of sequence n: [lo, hi) of the packed tensors or of its own rows.  Whatever the offsets hold, 0 <= lo <= hi <= rows.
__device__ __forceinline__ void row_range(const int32_t *offsets, int rows, int n, int &lo, int &hi) {
    lo = 0;
    hi = rows;
    if (offsets) {
        lo = min(max(offsets[n], 0), rows);
        hi = min(max(offsets[n + 1], lo), rows);
    }
}

template <typename T> __device__ __forceinline__ const T *row_ptr(const View &t, int packed, int n, int h, int row) {
    return (const T *)t.p + (packed ? 0 : n * t.seq) + row * t.row + (h / t.share) * t.head;
}

// The recurrence one row at a time: a workgroup per (sequence, head), a thread holds half a column of the state.
template <typename T, bool TANGENT>
__global__ __launch_bounds__(256) void td_decay_serial_kernel(Pass P) {
    constexpr int D = TD_DECAY_MAX_DIM, HALF = D / 2;
    __shared__ float sa[D], sb[D], sc[D], part[2][D];
    __shared__ double red[256];
    const int h = blockIdx.x % P.heads, n = blockIdx.x / P.heads, tid = threadIdx.x;
    const int col = tid & (D - 1), half = tid / D, packed = P.offsets != nullptr;
    int lo, hi;
    row_range(P.offsets, P.rows, n, lo, hi);
    const float g = expf(P.log_decay[h]);
    const int64_t state_at = ((int64_t)n * P.heads + h) * P.da * P.dc;
    float S[HALF], H[TANGENT ? HALF : 1];
#pragma unroll
    for (int r = 0; r < HALF; ++r) {
        const int i = half * HALF + r;
        S[r] = P.state_in && i < P.da && col < P.dc ? P.state_in[state_at + i * P.st_a + col * P.st_c] : 0.0f;
        if (TANGENT) H[r] = 0.0f;
    }
    double slope = 0.0;
    for (int t = 0; t < hi - lo; ++t) {
        const int row = P.reverse ? hi - 1 - t : lo + t;
        __syncthreads();
        if (tid < D) {
            sa[tid] = tid < P.da ? as_float<T>(row_ptr<T>(P.a, packed, n, h, row)[tid]) : 0.0f;
            sb[tid] = tid < P.da ? as_float<T>(row_ptr<T>(P.b, packed, n, h, row)[tid]) : 0.0f;
        } else {
            sc[col] = col < P.dc ? as_float<T>(row_ptr<T>(P.c, packed, n, h, row)[col]) : 0.0f;
        }
        __syncthreads();
        const float c = sc[col] * P.upd_scale;
        float sum = 0.0f, tan = 0.0f;
#pragma unroll
        for (int r = 0; r < HALF; ++r) {
            const float a = sa[half * HALF + r], b = sb[half * HALF + r];
            if (P.reverse) {
                S[r] += b * c;
                sum += a * S[r];
                S[r] *= g;
            } else {
                if (TANGENT) {
                    H[r] = g * (H[r] + S[r]);
                    tan += a * H[r];
                }
                S[r] = g * S[r] + b * c;
                sum += a * S[r];
            }
        }
        part[half][col] = sum;
        __syncthreads();
        const int64_t at = ((int64_t)(packed ? 0 : n) * P.rows + row) * P.heads + h;
        if (half == 0 && col < P.dc && P.out) {
            const float v = (part[0][col] + part[1][col]) * P.out_scale;
            if (P.out_f32) ((float *)P.out)[at * P.dc + col] = v;
            else ((T *)P.out)[at * P.dc + col] = (T)v;
        }
        if (TANGENT && col < P.dc) slope += (double)(tan * P.out_scale * as_float<T>(row_ptr<T>(P.e, packed, n, h, row)[col]));
    }
#pragma unroll
    for (int r = 0; r < HALF; ++r) {
        const int i = half * HALF + r;
        if (i < P.da && col < P.dc) {
            const int64_t at = state_at + i * P.st_a + col * P.st_c;
            if (P.state_out) P.state_out[at] = S[r];
            if (TANGENT && P.grad_state) slope += (double)(H[r] * P.grad_state[at]);
        }
    }
    if (TANGENT) {
        red[tid] = slope;
        __syncthreads();
        for (int o = 128; o > 0; o >>= 1) {
            if (tid < o) red[tid] += red[tid + o];
            __syncthreads();
        }
        if (tid == 0) P.slope[blockIdx.x] = red[0];
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
        const T *a = row_ptr<T>(P.a, 0, n, h, 0), *b = row_ptr<T>(P.b, 0, n, h, 0);
        const float c = as_float<T>(row_ptr<T>(P.c, 0, n, h, 0)[col]);
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
    TD_REQUIRE((int64_t)c->n_seq * c->heads <= (1 << 30), "n_seq * heads must be at most 2^30");
    return TD_OK;
}

int64_t total_rows(const td_decay_config *c) { return c->packed ? c->rows : (int64_t)c->n_seq * c->rows; }
size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

View view(const void *p, const int64_t *s, int heads, int own) { return View{p, s[0], s[1], s[2], heads / own}; }

Pass base_pass(const td_decay_config *c, const float *log_decay, const int32_t *offsets) {
    Pass P = {};
    P.log_decay = log_decay;
    P.offsets = c->packed ? offsets : nullptr;
    P.n_seq = c->n_seq;
    P.rows = c->rows;
    P.heads = c->heads;
    P.out_scale = P.upd_scale = 1.0f;
    return P;
}

template <bool TANGENT> int launch_pass(const td_decay_config *c, const Pass &P, hipStream_t st) {
    const dim3 grid(c->n_seq * c->heads);
    if (c->dtype == TD_BF16) hipLaunchKernelGGL((td_decay_serial_kernel<__bf16, TANGENT>), grid, dim3(256), 0, st, P);
    else hipLaunchKernelGGL((td_decay_serial_kernel<float, TANGENT>), grid, dim3(256), 0, st, P);
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
    int rc = tangent ? launch_pass<true>(c, P, st) : launch_pass<false>(c, P, st);
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

struct Layout { size_t slope, parts, total; };
Layout backward_layout(const td_decay_config *c) {
    Layout w;
    w.slope = 0;
    w.parts = up256((size_t)c->n_seq * c->heads * sizeof(double));
    const int d = c->dk > c->dv ? c->dk : c->dv;
    const bool shared = c->q_heads != c->heads || c->k_heads != c->heads || c->v_heads != c->heads;
    w.total = w.parts + (shared ? up256((size_t)total_rows(c) * c->heads * d * sizeof(float)) : 0);
    return w;
}

}  // namespace

extern "C" size_t td_decay_workspace_bytes(const td_decay_config *cfg, int32_t backward) {
    if (check_config(cfg) != TD_OK) return 0;
    return backward ? backward_layout(cfg).total : 256;
}

extern "C" int td_decay_forward(const td_decay_config *cfg, const void *q, const void *k, const void *v, const float *log_decay,
                                const int32_t *offsets, const float *state_in, void *o, float *state_out, void *workspace, void *stream) {
    if (int rc = check_config(cfg)) return rc;
    TD_REQUIRE(log_decay && workspace && (cfg->rows == 0 || (q && k && v && o)), "null pointer");
    TD_REQUIRE(!cfg->packed || offsets, "packed sequences need offsets");
    TD_REQUIRE(!state_out || state_out != state_in, "state_in and state_out must not be the same memory");
    Pass P = base_pass(cfg, log_decay, offsets);
    P.a = view(q, cfg->q_stride, cfg->heads, cfg->q_heads);
    P.b = view(k, cfg->k_stride, cfg->heads, cfg->k_heads);
    P.c = view(v, cfg->v_stride, cfg->heads, cfg->v_heads);
    P.da = cfg->dk; P.dc = cfg->dv; P.st_a = cfg->dv; P.st_c = 1;
    P.state_in = state_in; P.state_out = state_out;
    P.out = o; P.out_scale = cfg->scale;
    if (int rc = launch_pass<false>(cfg, P, (hipStream_t)stream)) return rc;
    return clear_rows(cfg, offsets, cfg->heads * cfg->dv, o, (hipStream_t)stream);
}

extern "C" int td_decay_backward(const td_decay_config *cfg, const void *q, const void *k, const void *v, const float *log_decay,
                                 const int32_t *offsets, const float *state_in, const void *grad_o, const float *grad_state_out, void *grad_q,
                                 void *grad_k, void *grad_v, float *grad_log_decay, float *grad_state_in, void *workspace, void *stream) {
    if (int rc = check_config(cfg)) return rc;
    TD_REQUIRE(log_decay && workspace && (cfg->rows == 0 || (q && k && v && grad_o)), "null pointer");
    TD_REQUIRE(!cfg->packed || offsets, "packed sequences need offsets");
    hipStream_t st = (hipStream_t)stream;
    const Layout w = backward_layout(cfg);
    float *parts = (float *)((char *)workspace + w.parts);
    const View vq = view(q, cfg->q_stride, cfg->heads, cfg->q_heads), vk = view(k, cfg->k_stride, cfg->heads, cfg->k_heads),
               vv = view(v, cfg->v_stride, cfg->heads, cfg->v_heads), vo = view(grad_o, cfg->grad_o_stride, cfg->heads, cfg->heads);
    if (grad_q || grad_log_decay) {
        Pass P = base_pass(cfg, log_decay, offsets);
        P.a = vo; P.b = vv; P.c = vk; P.e = vq;
        P.da = cfg->dv; P.dc = cfg->dk; P.st_a = 1; P.st_c = cfg->dv;
        P.state_in = state_in; P.grad_state = grad_state_out; P.slope = (double *)((char *)workspace + w.slope);
        P.out_scale = cfg->scale;
        if (int rc = grad_pass(cfg, P, cfg->q_heads, cfg->dk, grad_q, parts, grad_log_decay != nullptr, st)) return rc;
        if (grad_log_decay) {
            hipLaunchKernelGGL(td_decay_slope_kernel, dim3(cfg->heads), dim3(256), 0, st, P.slope, cfg->n_seq, cfg->heads, grad_log_decay);
            TD_LAUNCH_CHECK();
        }
    }
    if (grad_v || grad_state_in) {
        Pass P = base_pass(cfg, log_decay, offsets);
        P.reverse = 1;
        P.a = vk; P.b = vq; P.c = vo;
        P.da = cfg->dk; P.dc = cfg->dv; P.st_a = cfg->dv; P.st_c = 1;
        P.state_in = grad_state_out; P.state_out = grad_state_in; P.upd_scale = cfg->scale;
        if (int rc = grad_pass(cfg, P, cfg->v_heads, cfg->dv, grad_v, parts, false, st)) return rc;
    }
    if (grad_k) {
        Pass P = base_pass(cfg, log_decay, offsets);
        P.reverse = 1;
        P.a = vv; P.b = vo; P.c = vq;
        P.da = cfg->dv; P.dc = cfg->dk; P.st_a = 1; P.st_c = cfg->dv;
        P.state_in = grad_state_out; P.upd_scale = cfg->scale;
        if (int rc = grad_pass(cfg, P, cfg->k_heads, cfg->dk, grad_k, parts, false, st)) return rc;
    }
    return TD_OK;
}

extern "C" int td_decay_step(const td_decay_config *cfg, const void *q, const void *k, const void *v, const float *log_decay, float *state,
                             void *o, void *stream) {
    if (int rc = check_config(cfg)) return rc;
    TD_REQUIRE(cfg->rows == 1 && !cfg->packed, "td_decay_step takes one row of each sequence (rows = 1, packed = 0)");
    TD_REQUIRE(q && k && v && log_decay && state && o, "null pointer");
    Pass P = base_pass(cfg, log_decay, nullptr);
    P.a = view(q, cfg->q_stride, cfg->heads, cfg->q_heads);
    P.b = view(k, cfg->k_stride, cfg->heads, cfg->k_heads);
    P.c = view(v, cfg->v_stride, cfg->heads, cfg->v_heads);
    P.da = cfg->dk; P.dc = cfg->dv;
    P.state_out = state; P.out = o; P.out_scale = cfg->scale;
    const dim3 grid(cfg->n_seq * cfg->heads);
    if (cfg->dtype == TD_BF16) hipLaunchKernelGGL(td_decay_step_kernel<__bf16>, grid, dim3(256), 0, (hipStream_t)stream, P);
    else hipLaunchKernelGGL(td_decay_step_kernel<float>, grid, dim3(256), 0, (hipStream_t)stream, P);
    TD_LAUNCH_CHECK();
    return TD_OK;
}
