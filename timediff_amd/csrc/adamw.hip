// AdamW over a list of tensors in one launch (include/timediff_hip.h), moments in 32 or in 8 bits.
//
// Bound by memory: 28 bytes a value with 32-bit moments (param, m, v read and written, grad read), 16 with 8-bit ones.  The list
// travels in the kernel's arguments (nothing is kept between calls and a graph captures it): a workgroup finds its tensor in a
// prefix sum of workgroup counts.  A wave steps one block of 256 values, four a lane: the block is what shares a scale, so
// its largest magnitude is a reduction inside the wave and the moments are read and written once.
#include "common.h"
#include "rng.h"

namespace {

constexpr int MAX_TENSORS = 48;      // records of one launch: 48 x 64 bytes of the 4 KiB of kernel arguments
constexpr int WAVES = 4;             // blocks of 256 values that a workgroup takes
constexpr int64_t MAX_GROUPS = 0xFFFFFFFFll / (64 * WAVES);      // HIP launches fewer than 2^32 threads at once

struct Batch {
    td_adamw_tensor t[MAX_TENSORS];  // .reserved: 1 where every pointer is aligned for four values at once
    int first[MAX_TENSORS + 1];      // workgroups before each tensor's own
    int count, position;             // records here; place of the first one in the caller's list
    int done;                        // workgroups of the first record that an earlier launch had
    float beta1, beta2, omb1, omb2, eps, step_size, inv_sqrt_bc2, decay;
    uint64_t seed;
    uint32_t step;
    const float *grad_scale;
    const td_adamw_record *rec;
};

struct Scalars { float step_size, inv_sqrt_bc2, decay; uint64_t seed; uint32_t step; };

// the decayed parameter is rounded before the subtraction (no fused multiply-add), as a multiplication of its own would be
__device__ __forceinline__ float decayed(float p, float decay) {
#pragma clang fp contract(off)
    return p * decay;
}

// The moments.  With 8-bit moments every operation is rounded on its own (no fused multiply-add): which neighbour a value goes to
// then follows from the formula in float32 alone, whoever computes it.
template <int BITS> __device__ __forceinline__ void moments(float &m, float &v, float g, float beta1, float beta2, float omb1, float omb2) {
    if (BITS == 8) {
#pragma clang fp contract(off)
        m = beta1 * m + omb1 * g;
        v = beta2 * v + omb2 * g * g;
    } else {
        m = beta1 * m + omb1 * g;
        v = beta2 * v + omb2 * g * g;
    }
}

// one of the two e4m3 neighbours of y in [0, 448]: t = y / (its binade's step) in [8, 16) (below 2^-6: [0, 8)), up where
// the fraction plus u in (0, 1) passes one
__device__ __forceinline__ uint32_t e4m3_round(float y, uint32_t bits16) {
#pragma clang fp contract(off)
    const float u = ((float)bits16 + 0.5f) * (1.0f / 65536.0f);
    int e = (int)(__float_as_uint(y) >> 23) - 127;
    e = e < -6 ? -6 : e;
    const float t = y * __uint_as_float((uint32_t)(130 - e) << 23);
    const int c = ((e + 7) << 3) - 8 + (int)floorf(t + u);
    return y != y ? 0x7Fu : (uint32_t)(c > 126 ? 126 : c);
}

// the block's largest magnitude, on the bit patterns: a NaN is larger than everything and stays
__device__ __forceinline__ float wave_top(float x) {
    uint32_t b = __float_as_uint(x);
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t other = __shfl_xor(b, o);
        b = other > b ? other : b;
    }
    return __uint_as_float(b);
}

__device__ __forceinline__ float load_grad(const td_adamw_tensor &t, int64_t i) {
    return t.grad_dtype == TD_BF16 ? (float)((const __bf16 *)t.grad)[i] : ((const float *)t.grad)[i];
}

template <int BITS>
__device__ __forceinline__ void step_block(const Batch &B, const Scalars &s, const td_adamw_tensor &t, int position, int64_t block, int lane, float gs) {
    const int64_t base = block * TD_ADAMW_BLOCK;
    const int left = t.n - base < TD_ADAMW_BLOCK ? (int)(t.n - base) : TD_ADAMW_BLOCK;
    const bool vec = t.reserved && left == TD_ADAMW_BLOCK;
    // aligned whole blocks: four neighbours a lane (16-byte accesses); else every 64th, so that a wave's accesses stay adjacent
    const int at = vec ? 4 * lane : lane, by = vec ? 1 : 64;
    float p[4], g[4], m[4], v[4];
    if (vec) {
        const f32x4 x = *(const f32x4 *)(t.param + base + at);
        for (int j = 0; j < 4; ++j) p[j] = x[j];
        if (t.grad_dtype == TD_BF16) {
            const uint2 y = *(const uint2 *)((const uint16_t *)t.grad + base + at);
            g[0] = __uint_as_float(y.x << 16); g[1] = __uint_as_float(y.x & 0xFFFF0000u);
            g[2] = __uint_as_float(y.y << 16); g[3] = __uint_as_float(y.y & 0xFFFF0000u);
        } else {
            const f32x4 y = *(const f32x4 *)((const float *)t.grad + base + at);
            for (int j = 0; j < 4; ++j) g[j] = y[j];
        }
    } else {
        for (int j = 0; j < 4; ++j) {
            const int i = at + j * by;
            p[j] = i < left ? t.param[base + i] : 0.0f;
            g[j] = i < left ? load_grad(t, base + i) : 0.0f;
        }
    }
    uint32_t mb = 0, vb = 0;
    if (BITS == 8) {
        const float sm = t.scales[2 * block], sv = t.scales[2 * block + 1];
        if (vec) {
            mb = *(const uint32_t *)((const uint8_t *)t.exp_avg + base + at);
            vb = *(const uint32_t *)((const uint8_t *)t.exp_avg_sq + base + at);
        } else {
            for (int j = 0; j < 4; ++j)
                if (at + j * by < left) {
                    mb |= (uint32_t)((const uint8_t *)t.exp_avg)[base + at + j * by] << (8 * j);
                    vb |= (uint32_t)((const uint8_t *)t.exp_avg_sq)[base + at + j * by] << (8 * j);
                }
        }
        m[0] = __builtin_amdgcn_cvt_f32_fp8(mb, 0) * sm; m[1] = __builtin_amdgcn_cvt_f32_fp8(mb, 1) * sm;
        m[2] = __builtin_amdgcn_cvt_f32_fp8(mb, 2) * sm; m[3] = __builtin_amdgcn_cvt_f32_fp8(mb, 3) * sm;
        v[0] = __builtin_amdgcn_cvt_f32_fp8(vb, 0) * sv; v[1] = __builtin_amdgcn_cvt_f32_fp8(vb, 1) * sv;
        v[2] = __builtin_amdgcn_cvt_f32_fp8(vb, 2) * sv; v[3] = __builtin_amdgcn_cvt_f32_fp8(vb, 3) * sv;
        for (int j = 0; j < 4; ++j) v[j] *= v[j];
    } else if (vec) {
        const f32x4 x = *(const f32x4 *)((const float *)t.exp_avg + base + at), y = *(const f32x4 *)((const float *)t.exp_avg_sq + base + at);
        for (int j = 0; j < 4; ++j) { m[j] = x[j]; v[j] = y[j]; }
    } else {
        for (int j = 0; j < 4; ++j) {
            const int i = at + j * by;
            m[j] = i < left ? ((const float *)t.exp_avg)[base + i] : 0.0f;
            v[j] = i < left ? ((const float *)t.exp_avg_sq)[base + i] : 0.0f;
        }
    }
    float root[4];
    for (int j = 0; j < 4; ++j) {
        g[j] = g[j] * gs;
        moments<BITS>(m[j], v[j], g[j], B.beta1, B.beta2, B.omb1, B.omb2);
        root[j] = sqrtf(v[j]);
        p[j] = decayed(p[j], s.decay) - s.step_size * m[j] / (root[j] * s.inv_sqrt_bc2 + B.eps);
    }
    if (vec) {
        *(f32x4 *)(t.param + base + at) = f32x4{p[0], p[1], p[2], p[3]};
    } else {
        for (int j = 0; j < 4; ++j)
            if (at + j * by < left) t.param[base + at + j * by] = p[j];
    }
    if (BITS == 32) {
        float *pm = (float *)t.exp_avg + base, *pv = (float *)t.exp_avg_sq + base;
        if (vec) {
            *(f32x4 *)(pm + at) = f32x4{m[0], m[1], m[2], m[3]};
            *(f32x4 *)(pv + at) = f32x4{v[0], v[1], v[2], v[3]};
        } else {
            for (int j = 0; j < 4; ++j)
                if (at + j * by < left) { pm[at + j * by] = m[j]; pv[at + j * by] = v[j]; }
        }
        return;
    }
    uint32_t rnd[4] = {0, 0, 0, 0};
    if (t.random) {
        if (vec) {
            const uint4 x = *(const uint4 *)(t.random + base + at);
            rnd[0] = x.x; rnd[1] = x.y; rnd[2] = x.z; rnd[3] = x.w;
        } else {
            for (int j = 0; j < 4; ++j) rnd[j] = at + j * by < left ? (uint32_t)t.random[base + at + j * by] : 0u;
        }
    } else {
        // value i takes word i % 4 of the Philox block (i / 4, position, step)
        const uint32_t k0 = (uint32_t)s.seed, k1 = (uint32_t)(s.seed >> 32);
        if (vec) {
            const uint64_t q = (uint64_t)(base + at) >> 2;
            const Philox4 x = td_philox((uint32_t)q, (uint32_t)(q >> 32), (uint32_t)position, s.step, k0, k1);
            for (int j = 0; j < 4; ++j) rnd[j] = x.v[j];
        } else {
            for (int j = 0; j < 4; ++j) {
                const uint64_t i = (uint64_t)(base + at + j * by), q = i >> 2;
                const Philox4 x = td_philox((uint32_t)q, (uint32_t)(q >> 32), (uint32_t)position, s.step, k0, k1);
                const int w = (int)(i & 3);
                rnd[j] = w == 0 ? x.v[0] : w == 1 ? x.v[1] : w == 2 ? x.v[2] : x.v[3];
            }
        }
    }
    float top_m = 0.0f, top_v = 0.0f;
    for (int j = 0; j < 4; ++j) {
        if (vec || at + j * by < left) {
            const uint32_t a = __float_as_uint(fabsf(m[j])), b = __float_as_uint(root[j]) & 0x7FFFFFFFu;
            top_m = a > __float_as_uint(top_m) ? __uint_as_float(a) : top_m;
            top_v = b > __float_as_uint(top_v) ? __uint_as_float(b) : top_v;
        }
    }
    top_m = wave_top(top_m);
    top_v = wave_top(top_v);
    const bool some_m = !(top_m < 0x1p-100f), some_v = !(top_v < 0x1p-100f);
    const float im = some_m ? 448.0f * (1.0f / top_m) : 0.0f, iv = some_v ? 448.0f * (1.0f / top_v) : 0.0f;
    mb = vb = 0;
    for (int j = 0; j < 4; ++j) {
        float ym = fabsf(m[j]) * im, yv = root[j] * iv;
        ym = ym > 448.0f ? 448.0f : ym;
        yv = yv > 448.0f ? 448.0f : yv;
        const uint32_t cm = e4m3_round(ym, rnd[j] & 0xFFFFu) | (__float_as_uint(m[j]) >> 31 << 7);
        uint32_t cv = e4m3_round(yv, rnd[j] >> 16);
        cv = cv == 0 && some_v && root[j] > 0.0f ? 1u : cv;
        mb |= cm << (8 * j);
        vb |= cv << (8 * j);
    }
    if (vec) {
        *(uint32_t *)((uint8_t *)t.exp_avg + base + at) = mb;
        *(uint32_t *)((uint8_t *)t.exp_avg_sq + base + at) = vb;
    } else {
        for (int j = 0; j < 4; ++j)
            if (at + j * by < left) {
                ((uint8_t *)t.exp_avg)[base + at + j * by] = (uint8_t)(mb >> (8 * j));
                ((uint8_t *)t.exp_avg_sq)[base + at + j * by] = (uint8_t)(vb >> (8 * j));
            }
    }
    if (lane == 0) {
        t.scales[2 * block] = some_m ? top_m * (1.0f / 448.0f) : 0.0f;
        t.scales[2 * block + 1] = some_v ? top_v * (1.0f / 448.0f) : 0.0f;
    }
}

template <int BITS> __global__ __launch_bounds__(64 * WAVES) void td_adamw_kernel(Batch B) {
    int lo = 0, hi = B.count - 1;        // the last tensor that begins at or before this workgroup
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (B.first[mid] <= (int)blockIdx.x) lo = mid;
        else hi = mid - 1;
    }
    const td_adamw_tensor &t = B.t[lo];
    Scalars s{B.step_size, B.inv_sqrt_bc2, B.decay, B.seed, B.step};
    if (B.rec) s = Scalars{B.rec->step_size, B.rec->inv_sqrt_bc2, B.rec->decay, B.rec->seed, (uint32_t)B.rec->step};
    const float gs = B.grad_scale ? B.grad_scale[0] : 1.0f;
    const int64_t block = (int64_t)(blockIdx.x - B.first[lo] + (lo == 0 ? B.done : 0)) * WAVES + threadIdx.x / 64;
    if (block * TD_ADAMW_BLOCK < t.n) step_block<BITS>(B, s, t, B.position + lo, block, threadIdx.x % 64, gs);
}

int check_config(const td_adamw_config *c) {
    TD_REQUIRE(c, "configuration required");
    TD_REQUIRE(c->step >= 1, "step counts from 1, got %lld", (long long)c->step);
    TD_REQUIRE(c->beta1 >= 0.0 && c->beta1 < 1.0 && c->beta2 >= 0.0 && c->beta2 < 1.0, "betas must be in [0, 1), got %g and %g", c->beta1, c->beta2);
    TD_REQUIRE(c->lr >= 0.0 && c->eps >= 0.0 && c->weight_decay >= 0.0, "lr, eps and weight_decay must not be negative");
    TD_REQUIRE(c->state_bits == 32 || c->state_bits == 8, "state_bits must be 32 or 8, got %d", c->state_bits);
    return TD_OK;
}

void step_values(const td_adamw_config *c, float &step_size, float &inv_sqrt_bc2, float &decay) {
    step_size = (float)(c->lr / (1.0 - pow(c->beta1, (double)c->step)));
    inv_sqrt_bc2 = (float)(1.0 / sqrt(1.0 - pow(c->beta2, (double)c->step)));
    decay = (float)(1.0 - c->lr * c->weight_decay);
}

bool aligned(const td_adamw_tensor &t, int bits) {
    const uintptr_t state = (uintptr_t)t.exp_avg | (uintptr_t)t.exp_avg_sq;
    return ((uintptr_t)t.param | (uintptr_t)t.random) % 16 == 0 && (uintptr_t)t.grad % (t.grad_dtype == TD_BF16 ? 8 : 16) == 0 &&
           state % (bits == 8 ? 4 : 16) == 0;
}

__global__ void td_adamw_record_kernel(td_adamw_record *dst, td_adamw_record v) { *dst = v; }

}  // namespace

extern "C" int td_adamw(const td_adamw_config *cfg, const td_adamw_tensor *tensors_host, int32_t count, void *stream) {
    if (int rc = check_config(cfg)) return rc;
    TD_REQUIRE(count >= 0 && (count == 0 || tensors_host), "bad tensor list");
    for (int i = 0; i < count; ++i) {
        const td_adamw_tensor &t = tensors_host[i];
        TD_REQUIRE(t.n >= 0, "tensor %d: bad size", i);
        TD_REQUIRE(t.n < (1LL << 40), "tensor %d: too large", i);
        TD_REQUIRE(t.n == 0 || (t.param && t.grad && t.exp_avg && t.exp_avg_sq), "tensor %d: null pointer", i);
        TD_REQUIRE(t.grad_dtype == TD_F32 || t.grad_dtype == TD_BF16, "tensor %d: gradients must be TD_F32 or TD_BF16, got %d", i, t.grad_dtype);
        TD_REQUIRE(t.n == 0 || cfg->state_bits == 32 || t.scales, "tensor %d: 8-bit moments need scales", i);
    }
    Batch B;
    B.beta1 = (float)cfg->beta1; B.beta2 = (float)cfg->beta2; B.omb1 = (float)(1.0 - cfg->beta1); B.omb2 = (float)(1.0 - cfg->beta2);
    B.eps = (float)cfg->eps;
    step_values(cfg, B.step_size, B.inv_sqrt_bc2, B.decay);
    B.seed = cfg->seed; B.step = (uint32_t)cfg->step; B.grad_scale = cfg->grad_scale; B.rec = cfg->record;
    B.done = 0;
    for (int i = 0; i < count;) {
        int64_t groups = 0;
        int left_off = 0;
        B.position = i;
        B.count = 0;
        while (i < count && B.count < MAX_TENSORS && groups < MAX_GROUPS) {
            const td_adamw_tensor &t = tensors_host[i];
            const int64_t done = B.count == 0 ? B.done : 0, mine = (t.n + TD_ADAMW_BLOCK * WAVES - 1) / (TD_ADAMW_BLOCK * WAVES) - done;
            B.t[B.count] = t;
            B.t[B.count].reserved = aligned(t, cfg->state_bits);
            B.first[B.count++] = (int)groups;
            if (groups + mine > MAX_GROUPS) {          // the next launch goes on inside this tensor
                left_off = (int)(done + MAX_GROUPS - groups);
                groups = MAX_GROUPS;
                break;
            }
            groups += mine;
            ++i;
        }
        if (groups == 0) continue;
        if (cfg->state_bits == 32) hipLaunchKernelGGL(td_adamw_kernel<32>, dim3((unsigned)groups), dim3(64 * WAVES), 0, (hipStream_t)stream, B);
        else hipLaunchKernelGGL(td_adamw_kernel<8>, dim3((unsigned)groups), dim3(64 * WAVES), 0, (hipStream_t)stream, B);
        TD_LAUNCH_CHECK();
        B.done = left_off;
    }
    return TD_OK;
}

extern "C" int td_adamw_record_set(td_adamw_record *record_dev, const td_adamw_config *cfg, void *stream) {
    if (int rc = check_config(cfg)) return rc;
    TD_REQUIRE(record_dev, "null pointer");
    td_adamw_record r;
    r.seed = cfg->seed;
    r.step = cfg->step;
    step_values(cfg, r.step_size, r.inv_sqrt_bc2, r.decay);
    r.reserved = 0.0f;
    hipLaunchKernelGGL(td_adamw_record_kernel, dim3(1), dim3(1), 0, (hipStream_t)stream, record_dev, r);   // the values travel as kernel arguments
    TD_LAUNCH_CHECK();
    return TD_OK;
}
