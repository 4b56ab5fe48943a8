// The chunked kernel of decay attention (decay_attn.hip has the formulas): a workgroup takes one sequence (or a segment of one) and
// head, 64 rows at a time, and keeps the state in registers between the chunks.  With i, j rows of a chunk of n, F the state
// entering it and X^T standing for a matrix with its columns in lanes,
//     out_i = os (g^(i+1) F^T a_i + sum_{j<=i} g^(i-j) (b_j . a_i) us c_j),       F' = g^n F + sum_j g^(n-1-j) us b_j c_j^T
// (reversed passes: out's exponent is one less, F's terms' one more).  Everything is 16 x 16 matrix tiles, and the order of an operand's
// inner index is free as long as both operands share it, so that no product's result is ever moved between lanes:
//   * a wave owns 16 CT columns of c and of the state; the state's accumulators (rows = da in a lane's registers, lane = column) ARE
//     the operand of F^T a, and the scores' accumulators (rows j in registers, lane = row i) the operand of the sum over j;
//   * b and c are read from LDS with rows as the inner index by transposing loads (ds_read_b64_tr_b16).
// bfloat16: v_mfma_f32_16x16x32_bf16, and an operand that is not an input is split into bf16 terms: scores and states
// into two (2^-17 of each, below what the output's own rounding leaves), decayed rows that enter the state, and everything behind a float32
// result, into three (2^-24).  float32: v_mfma_f32_16x16x4_f32.
#pragma once
#include "common.h"

namespace decay {

constexpr int CHUNK = 64;

struct View {                 // rows of one tensor; head h of the recurrence reads head h / share
    const void *p;
    int64_t seq, row, head;
    int share, d, vec;        // vec: 16-byte loads fit
};

struct Pass {
    View a, b, c, e;          // e: what the tangent's output is dotted with (tangent form only)
    const float *log_decay;
    const int32_t *offsets;   // packed: n_seq + 1, else NULL
    const float *state_in;    // (n_seq, heads, ..): element (i, j) of (da, dc) at i * st_a + j * st_c, NULL: zeros
    float *state_out;         // NULL: not wanted
    const float *grad_state;  // tangent form: the gradient of the state left behind, NULL: none
    float *seg, *seg_tan;     // (slots, heads, ..) as state_in: the state (its tangent) entering each segment; SUM form: what each one adds
    double *slope;            // tangent form: one sum for each (slot, head)
    int64_t st_a, st_c;
    void *out;                // (rows, heads, dc), float32 (out_f32) or the tensors' type; NULL: not wanted
    int out_f32, out_vec;
    int n_seq, rows, heads, da, dc, reverse;
    int seg_len, segs, slots; // rows of a segment (a multiple of CHUNK), segments of a dense sequence (1: seg_len covers all), slots in all
    float out_scale, upd_scale;
};

// The rows of sequence n: [lo, hi) of the packed tensors or of its own rows.  Whatever the offsets hold, 0 <= lo <= hi <= rows.
__device__ __forceinline__ void row_range(const int32_t *offsets, int rows, int n, int &lo, int &hi) {
    lo = 0;
    hi = rows;
    if (offsets) {
        lo = min(max(offsets[n], 0), rows);
        hi = min(max(offsets[n + 1], lo), rows);
    }
}

// Packed sequence n owns the slots from lo(n) / seg_len + n on: a sequence of any length has as many as it has segments (one at least), no
// two share one, and there are rows / seg_len + n_seq in all, whatever the lengths are.
__device__ __forceinline__ int first_slot(const Pass &P, int n) { return min(max(P.offsets[n], 0), P.rows) / P.seg_len + n; }

// -> the sequence and segment of a slot; segment < 0 where it has none
__device__ __forceinline__ void slot_owner(const Pass &P, int slot, int &n, int &segment) {
    if (!P.offsets || P.segs == 1) {
        n = slot / P.segs;
        segment = slot % P.segs;
        return;
    }
    int lo = 0, hi = P.n_seq - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first_slot(P, mid) <= slot) lo = mid;
        else hi = mid - 1;
    }
    n = lo;
    segment = slot - first_slot(P, lo);
}

// g^e for a whole number e: 1 for e = 0, also where log g is -inf
__device__ __forceinline__ float power(float lg2, int e) { return e == 0 ? 1.0f : exp2f(lg2 * (float)e); }

template <typename T> struct Mat;
template <> struct Mat<__bf16> {
    typedef bf16x8 Op;
    static constexpr int KT = 2;        // tiles of 16 that an operand spans
    static constexpr int VEC = 8;       // elements of 16 bytes
    static constexpr bool SPLIT = true;
    static __device__ __forceinline__ f32x4 mma(Op a, Op b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    // columns are stored in the order of the inner index: of each 32, group g's four of the first 16, then its four of the second
    static __device__ __forceinline__ int place(int four) { return (four >> 3) * 32 + (four & 3) * 8 + ((four >> 2) & 1) * 4; }
    static __device__ __forceinline__ Op row_op(const __bf16 *t, int ld, int row, int ks, int g) { return *(const Op *)(t + row * ld + ks * 32 + g * 8); }
    static __device__ __forceinline__ Op col_op(const __bf16 *t, int ld, int tile, int kr, int g, int li) {
        typedef __attribute__((__vector_size__(4 * sizeof(short)))) short s16x4;
        typedef __attribute__((address_space(3))) s16x4 *lds;
        const __bf16 *p = t + (kr * 32 + g * 4 + (li >> 2)) * ld + place(tile * 4 + (li & 3));
        union { s16x4 s[2]; Op o; } x;
        x.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(void *)p);
        x.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(void *)(p + 16 * ld));
        return x.o;
    }
    // the operand whose elements are x[tile][register]
    template <int N> static __device__ __forceinline__ void split(const f32x4 *x, Op *p) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float v = x[j >> 2][j & 3];
#pragma unroll
            for (int k = 0; k < N; ++k) {
                p[k][j] = (__bf16)v;
                v -= (float)p[k][j];
            }
        }
    }
    static __device__ __forceinline__ float elem(Op o, int tile, int r) { return (float)o[tile * 4 + r]; }
};
template <> struct Mat<float> {
    typedef f32x4 Op;
    static constexpr int KT = 1, VEC = 4;
    static constexpr bool SPLIT = false;
    static __device__ __forceinline__ f32x4 mma(Op a, Op b, f32x4 c) {
#pragma unroll
        for (int r = 0; r < 4; ++r) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], b[r], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ int place(int four) { return four * 4; }
    static __device__ __forceinline__ Op row_op(const float *t, int ld, int row, int ks, int g) { return *(const Op *)(t + row * ld + ks * 16 + g * 4); }
    static __device__ __forceinline__ Op col_op(const float *t, int ld, int tile, int kr, int g, int li) {
        const float *p = t + (kr * 16 + g * 4) * ld + tile * 16 + li;
        return Op{p[0], p[ld], p[2 * ld], p[3 * ld]};
    }
    template <int N> static __device__ __forceinline__ void split(const f32x4 *x, Op *p) { p[0] = x[0]; }
    static __device__ __forceinline__ float elem(Op o, int, int r) { return o[r]; }
};

// One chunk's rows of one tensor on their way from memory to LDS, 16 bytes a piece
template <typename T, int DP, int NT> struct Stage {
    static constexpr int VEC = Mat<T>::VEC, PIECES = DP / VEC, N = CHUNK * PIECES / NT, LD = DP + VEC;
    uint4 r[N];
    __device__ __forceinline__ void load(const T *base, const View &v, int first, int step, int n, int tid) {
#pragma unroll
        for (int c = 0; c < N; ++c) {
            const int i = tid + c * NT, row = i / PIECES, col = i % PIECES * VEC;
            r[c] = uint4{0, 0, 0, 0};
            if (row < n && col < v.d) {
                const T *p = base + (int64_t)(first + step * row) * v.row + col;
                if (v.vec) {
                    r[c] = *(const uint4 *)p;
                } else {
                    union { uint4 u; T t[VEC]; } x;
                    x.u = r[c];
#pragma unroll
                    for (int j = 0; j < VEC; ++j)
                        if (col + j < v.d) x.t[j] = p[j];
                    r[c] = x.u;
                }
            }
        }
    }
    __device__ __forceinline__ void store(T *lds, int tid) const {
#pragma unroll
        for (int c = 0; c < N; ++c) {
            const int i = tid + c * NT, row = i / PIECES, piece = i % PIECES;
            if constexpr (VEC == 8) {
                *(uint2 *)(lds + row * LD + Mat<T>::place(2 * piece)) = uint2{r[c].x, r[c].y};
                *(uint2 *)(lds + row * LD + Mat<T>::place(2 * piece + 1)) = uint2{r[c].z, r[c].w};
            } else {
                *(uint4 *)(lds + row * LD + Mat<T>::place(piece)) = r[c];
            }
        }
    }
};

template <typename T> __device__ __forceinline__ const T *base_of(const View &v, bool packed, int n, int h) {
    return (const T *)v.p + (packed ? 0 : n * v.seq) + (h / v.share) * v.head;
}

// DP: da and dc padded to 32, 64 or 128.  NW waves of CT column tiles: NW * CT * 16 = DP.  TAN: with the derivative by log g carried
// beside the state.  SUM: no output, only what a segment adds to the state.
template <typename T, int DP, int NW, int CT, bool TAN, bool SUM> __global__ __launch_bounds__(64 * NW) void td_decay_chunk_kernel(Pass P) {
    typedef Mat<T> M;
    typedef typename M::Op Op;
    constexpr int NT = 64 * NW, LD = DP + M::VEC, TILES = DP / 16, KS = TILES / M::KT, RT = CHUNK / 16, KR = RT / M::KT;
    constexpr int S2 = M::SPLIT ? (TAN ? 3 : 2) : 1, S3 = M::SPLIT ? 3 : 1;
    static_assert(NW * CT == TILES, "every column tile has a wave");
    __shared__ __align__(16) T lds[(SUM ? 2 : TAN ? 4 : 3) * CHUNK * LD];
    T *const lb = lds, *const lc = lds + CHUNK * LD, *const la = lds + (SUM ? 0 : 2) * CHUNK * LD, *const le = lds + (TAN && !SUM ? 3 : 0) * CHUNK * LD;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, g = lane >> 4, li = lane & 15;
    const int h = blockIdx.x % P.heads, slot = blockIdx.x / P.heads;
    const bool packed = P.offsets != nullptr;
    int n_seq, segment, lo, hi;
    slot_owner(P, slot, n_seq, segment);
    row_range(P.offsets, P.rows, n_seq, lo, hi);
    const int len = hi - lo, t0 = segment * P.seg_len;
    if (segment < 0 || (segment > 0 && t0 >= len)) {
        if (TAN && !SUM && tid == 0) P.slope[blockIdx.x] = 0.0;
        return;
    }
    const bool last = len - t0 <= P.seg_len;
    if (SUM && last) return;
    const int t1 = last ? len : t0 + P.seg_len;
    const int step = P.reverse ? -1 : 1, origin = P.reverse ? hi - 1 : lo;      // row t of the recurrence is row origin + step * t
    const T *pa = base_of<T>(P.a, packed, n_seq, h), *pb = base_of<T>(P.b, packed, n_seq, h), *pc = base_of<T>(P.c, packed, n_seq, h);
    const T *pe = TAN && !SUM ? base_of<T>(P.e, packed, n_seq, h) : nullptr;

    const float ld = P.log_decay[h], lg2 = ld * 1.44269504f;
    const int late = P.reverse ? 1 : 0;
    // g^64 as two floats: it multiplies the state once a chunk, and its own rounding would add up over a long memory
    const double whole_d = exp((double)ld * CHUNK);
    const float whole = (float)whole_d, whole_lo = isinf(whole) || whole == 0.0f ? 0.0f : (float)(whole_d - (double)whole);
    float wa[RT][4], wu[RT][4], wo[RT];          // g^(i-j) by how many tiles apart; what row j of a full chunk enters the state with; g^(i+1)
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        wo[t] = power(lg2, t * 16 + li + 1 - late);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int apart = t * 16 + li - (g * 4 + r);
            wa[t][r] = apart < 0 ? 0.0f : power(lg2, apart);
            wu[t][r] = power(lg2, CHUNK - 1 - (t * 16 + g * 4 + r) + late) * P.upd_scale;
        }
    }

    f32x4 S[TILES][CT], H[TAN ? TILES : 1][CT];
    const int64_t state_at = ((int64_t)n_seq * P.heads + h) * P.da * P.dc, seg_at = (int64_t)blockIdx.x * P.da * P.dc;
    const float *enter = SUM ? nullptr : segment > 0 ? P.seg + seg_at : P.state_in ? P.state_in + state_at : nullptr;
    const float *enter_tan = TAN && !SUM && segment > 0 ? P.seg_tan + seg_at : nullptr;
#pragma unroll
    for (int mt = 0; mt < TILES; ++mt)
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = mt * 16 + g * 4 + r, j = (wave * CT + ct) * 16 + li;
                const bool there = i < P.da && j < P.dc;
                S[mt][ct][r] = there && enter ? enter[i * P.st_a + j * P.st_c] : 0.0f;
                if (TAN) H[mt][ct][r] = there && enter_tan ? enter_tan[i * P.st_a + j * P.st_c] : 0.0f;
            }

    Stage<T, DP, NT> sa, sb, sc, se;
    const auto fetch = [&](int t) {
        const int n = min(CHUNK, t1 - t), first = origin + step * t;
        sb.load(pb, P.b, first, step, n, tid);
        sc.load(pc, P.c, first, step, n, tid);
        if (!SUM) sa.load(pa, P.a, first, step, n, tid);
        if (TAN && !SUM) se.load(pe, P.e, first, step, n, tid);
    };
    double slope = 0.0;
    if (t0 < t1) fetch(t0);
    for (int t = t0; t < t1; t += CHUNK) {
        const int n = min(CHUNK, t1 - t);
        sb.store(lb, tid);
        sc.store(lc, tid);
        if (!SUM) sa.store(la, tid);
        if (TAN && !SUM) se.store(le, tid);
        __syncthreads();
        if (t + CHUNK < t1) fetch(t + CHUNK);

        Op vt[CT][KR];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int kr = 0; kr < KR; ++kr) vt[ct][kr] = M::col_op(lc, LD, wave * CT + ct, kr, g, li);

        if constexpr (!SUM) {
            f32x4 o[RT][CT], x[TAN ? RT : 1][CT];
#pragma unroll
            for (int it = 0; it < RT; ++it)
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) {
                    o[it][ct] = f32x4{0, 0, 0, 0};
                    if (TAN) x[it][ct] = f32x4{0, 0, 0, 0};
                }
            // F^T a
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) {
                    f32x4 part[M::KT];
                    Op f[S2], ft[TAN ? S2 : 1];
#pragma unroll
                    for (int k = 0; k < M::KT; ++k) part[k] = S[s * M::KT + k][ct];
                    M::template split<S2>(part, f);
                    if constexpr (TAN) {
#pragma unroll
                        for (int k = 0; k < M::KT; ++k) part[k] = H[s * M::KT + k][ct];
                        M::template split<S2>(part, ft);
                    }
#pragma unroll
                    for (int it = 0; it < RT; ++it) {
                        const Op q = M::row_op(la, LD, it * 16 + li, s, g);
#pragma unroll
                        for (int k = 0; k < S2; ++k) {
                            o[it][ct] = M::mma(f[k], q, o[it][ct]);
                            if constexpr (TAN) x[it][ct] = M::mma(ft[k], q, x[it][ct]);
                        }
                    }
                }
            // their weights, and the rows of this chunk
            float dot = 0.0f;
#pragma unroll
            for (int it = 0; it < RT; ++it) {
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) {
                    if constexpr (TAN) x[it][ct] = (x[it][ct] + o[it][ct] * (float)(it * 16 + li + 1)) * wo[it];
                    o[it][ct] = o[it][ct] * wo[it];
                }
                Op q[KS];
#pragma unroll
                for (int s = 0; s < KS; ++s) q[s] = M::row_op(la, LD, it * 16 + li, s, g);
#pragma unroll
                for (int kr = 0; kr <= it / M::KT; ++kr) {
                    f32x4 w[M::KT], wx[M::KT];
#pragma unroll
                    for (int k = 0; k < M::KT; ++k) {
                        const int jt = kr * M::KT + k;
                        f32x4 s4 = f32x4{0, 0, 0, 0};
                        if (jt <= it) {
#pragma unroll
                            for (int s = 0; s < KS; ++s) s4 = M::mma(M::row_op(lb, LD, jt * 16 + li, s, g), q[s], s4);
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const int apart = (it - jt) * 16 + li - (g * 4 + r);
                                s4[r] = apart >= 0 ? s4[r] * wa[it - jt][r] * P.upd_scale : 0.0f;
                                if (TAN) wx[k][r] = s4[r] * (float)apart;
                            }
                        } else if (TAN) {
                            wx[k] = s4;
                        }
                        w[k] = s4;
                    }
                    Op f[S2];
                    M::template split<S2>(w, f);
#pragma unroll
                    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                        for (int k = 0; k < S2; ++k) o[it][ct] = M::mma(vt[ct][kr], f[k], o[it][ct]);
                    if constexpr (TAN) {
                        M::template split<S2>(wx, f);
#pragma unroll
                        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                            for (int k = 0; k < S2; ++k) x[it][ct] = M::mma(vt[ct][kr], f[k], x[it][ct]);
                    }
                }
                const int i = it * 16 + li;
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) {
                    const int tile = wave * CT + ct, col = tile * 16 + g * 4;
                    if constexpr (TAN) {
                        const T *e = le + i * LD + M::place(tile * 4 + g);
#pragma unroll
                        for (int r = 0; r < 4; ++r) dot += x[it][ct][r] * (float)e[r];
                    }
                    if (P.out && i < n) {
                        const int64_t at = ((int64_t)(packed ? 0 : n_seq) * P.rows + origin + step * (t + i)) * P.heads + h;
                        const f32x4 v = o[it][ct] * P.out_scale;
                        if (P.out_f32) {
                            float *to = (float *)P.out + at * P.dc + col;
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                if (col + r < P.dc) to[r] = v[r];
                        } else {
                            T *to = (T *)P.out + at * P.dc + col;
                            union { T t[4]; uint2 u2; uint4 u4; } y;
#pragma unroll
                            for (int r = 0; r < 4; ++r) y.t[r] = (T)v[r];
                            if (P.out_vec) {
                                if (col < P.dc) {
                                    if constexpr (sizeof(T) == 2) *(uint2 *)to = y.u2;
                                    else *(uint4 *)to = y.u4;
                                }
                            } else {
#pragma unroll
                                for (int r = 0; r < 4; ++r)
                                    if (col + r < P.dc) to[r] = y.t[r];
                            }
                        }
                    }
                }
            }
            if (TAN) slope += (double)(dot * P.out_scale);
        }

        // F' = g^n F + sum_j g^(n-1-j) b_j c_j^T
        float decay = whole, decay_lo = whole_lo;
        if (n < CHUNK) {
            decay = power(lg2, n);
            decay_lo = 0.0f;
#pragma unroll
            for (int jt = 0; jt < RT; ++jt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int j = jt * 16 + g * 4 + r;
                    wu[jt][r] = j < n ? power(lg2, n - 1 - j + late) * P.upd_scale : 0.0f;
                }
        }
#pragma unroll
        for (int mt = 0; mt < TILES; ++mt)
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if (TAN) {
                        const float y = H[mt][ct][r] + (float)n * S[mt][ct][r];
                        H[mt][ct][r] = decay * y + decay_lo * y;
                    }
                    S[mt][ct][r] = decay * S[mt][ct][r] + decay_lo * S[mt][ct][r];
                }
#pragma unroll
        for (int kr = 0; kr < KR; ++kr) {
            Op u[CT][S3], ux[TAN ? CT : 1][S3];
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                f32x4 y[M::KT], z[M::KT];
#pragma unroll
                for (int k = 0; k < M::KT; ++k)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int j = (kr * M::KT + k) * 16 + g * 4 + r;
                        y[k][r] = M::elem(vt[ct][kr], k, r) * wu[kr * M::KT + k][r];
                        z[k][r] = y[k][r] * (float)(n - 1 - j);
                    }
                M::template split<S3>(y, u[ct]);
                if constexpr (TAN) M::template split<S3>(z, ux[ct]);
            }
#pragma unroll
            for (int mt = 0; mt < TILES; ++mt) {
                const Op b = M::col_op(lb, LD, mt, kr, g, li);
#pragma unroll
                for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                    for (int k = 0; k < S3; ++k) {
                        S[mt][ct] = M::mma(b, u[ct][k], S[mt][ct]);
                        if constexpr (TAN) H[mt][ct] = M::mma(b, ux[ct][k], H[mt][ct]);
                    }
            }
        }
        __syncthreads();
    }

    float *leave = SUM ? P.seg + seg_at : last && P.state_out ? P.state_out + state_at : nullptr;
    float *leave_tan = TAN && SUM ? P.seg_tan + seg_at : nullptr;
    const float *grad = TAN && !SUM && last && P.grad_state ? P.grad_state + state_at : nullptr;
#pragma unroll
    for (int mt = 0; mt < TILES; ++mt)
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = mt * 16 + g * 4 + r, j = (wave * CT + ct) * 16 + li;
                if (i >= P.da || j >= P.dc) continue;
                const int64_t at = i * P.st_a + j * P.st_c;
                if (leave) leave[at] = S[mt][ct][r];
                if (TAN && leave_tan) leave_tan[at] = H[mt][ct][r];
                if (TAN && grad) slope += (double)(H[mt][ct][r] * grad[at]);
            }
    if constexpr (TAN && !SUM) {
        __shared__ double red[NT];
        red[tid] = slope;
        __syncthreads();
        for (int o = NT / 2; o > 0; o >>= 1) {
            if (tid < o) red[tid] += red[tid + o];
            __syncthreads();
        }
        if (tid == 0) P.slope[blockIdx.x] = red[0];
    }
}

}  // namespace decay
