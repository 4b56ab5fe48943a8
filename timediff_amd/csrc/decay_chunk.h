// The chunked kernel of decay attention (decay_attn.hip has the formulas): a workgroup takes one sequence (or a segment of one) and
// head, 64 rows at a time, and keeps the state in registers between the chunks.  With i, j rows of a chunk of n, F the state
// entering it and X^T standing for a matrix with its columns in lanes,
//     out_i = os (g^(i+1) F^T a_i + sum_{j<=i} g^(i-j) (b_j . a_i) us c_j),       F' = g^n F + sum_j g^(n-1-j) us b_j c_j^T
// (reversed passes: out's exponent is one less, F's terms' one more).  Everything is 16 x 16 matrix tiles, and the order of an operand's
// inner index is free as long as both operands share it, so that no product's result is ever moved between lanes:
//   * a wave owns 16 CT columns of c and of the state; the state's accumulators (rows = da in a lane's registers, lane = column) ARE
//     the operand of F^T a, and the scores' accumulators (rows j in registers, lane = row i) the operand of the sum over j: the waves
//     share out the ten score tiles on and below the diagonal and pass them on through LDS as operands, lane by lane;
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
    int share, d;
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
    int out_f32;
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
__device__ __forceinline__ float power(float lg2, int e) { return e == 0 ? 1.0f : __builtin_amdgcn_exp2f(lg2 * (float)e); }

typedef __attribute__((__vector_size__(4 * sizeof(__bf16)))) __bf16 bf16x4;

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
    // one tile's terms into its half of the operands at to, to + 64, ..
    template <int N> static __device__ __forceinline__ void keep(f32x4 x, Op *to, int half) {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            bf16x4 y;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                y[r] = (__bf16)x[r];
                x[r] -= (float)y[r];
            }
            *((bf16x4 *)(to + 64 * k) + half) = y;
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
    template <int N> static __device__ __forceinline__ void keep(f32x4 x, Op *to, int) { *to = x; }
    static __device__ __forceinline__ float elem(Op o, int, int r) { return o[r]; }
};

// One chunk's rows of one tensor on their way from memory to LDS.  Memory is read in the order of its rows (n of them from `low` on), a
// reversed pass turns them round in LDS.  VEC: 16 bytes a load, at 32-bit offsets from the chunk's first row, into registers that are filled
// while the chunk before it is computed; else (odd sizes, strides or addresses) element by element when the chunk begins.
template <typename T, int DP, int NT, bool VEC> struct Stage {
    static constexpr int PER = Mat<T>::VEC, PIECES = DP / PER, N = VEC ? CHUNK * PIECES / NT : 1, LD = DP + PER;
    static_assert(NT % PIECES == 0, "a thread's pieces share their columns");
    uint4 r[N];
    uint32_t at;              // byte offset of the first piece; the others are whole rows further on
    __device__ __forceinline__ void init(const View &v, int tid) {
        at = (uint32_t)(tid / PIECES) * (uint32_t)(v.row * sizeof(T)) + tid % PIECES * 16;
#pragma unroll
        for (int c = 0; c < N; ++c) r[c] = uint4{0, 0, 0, 0};
    }
    template <bool FULL> __device__ __forceinline__ void load(const T *base, const View &v, int low, int n, int tid) {
        if (!VEC || tid % PIECES * PER >= v.d) return;
        const char *p = (const char *)(base + (int64_t)low * v.row);
        const int64_t by = NT / PIECES * v.row * (int64_t)sizeof(T);
#pragma unroll
        for (int c = 0; c < N; ++c) {
            if (!FULL) r[c] = uint4{0, 0, 0, 0};
            if (FULL || (tid + c * NT) / PIECES < n) r[c] = *(const uint4 *)(p + c * by + at);
        }
    }
    template <bool FULL> __device__ __forceinline__ void store(T *lds, const T *base, const View &v, int low, int n, int reverse, int tid) const {
        if (!VEC) {
            const T *p = base + (int64_t)low * v.row;
#pragma unroll 4
            for (int i = tid; i < CHUNK * DP; i += NT) {
                const int row = i / DP, col = i % DP, to = reverse && row < n ? n - 1 - row : row;
                lds[to * LD + Mat<T>::place(col >> 2) + (col & 3)] = row < n && col < v.d ? p[row * v.row + col] : (T)0.0f;
            }
            return;
        }
#pragma unroll
        for (int c = 0; c < N; ++c) {
            const int i = tid + c * NT, row = i / PIECES, piece = i % PIECES, to = reverse && (FULL || row < n) ? (FULL ? CHUNK : n) - 1 - row : row;
            if constexpr (PER == 8) {
                *(uint2 *)(lds + to * LD + Mat<T>::place(2 * piece)) = uint2{r[c].x, r[c].y};
                *(uint2 *)(lds + to * LD + Mat<T>::place(2 * piece + 1)) = uint2{r[c].z, r[c].w};
            } else {
                *(uint4 *)(lds + to * LD + Mat<T>::place(piece)) = r[c];
            }
        }
    }
};

template <typename T> __device__ __forceinline__ const T *base_of(const View &v, bool packed, int n, int h) {
    return (const T *)v.p + (packed ? 0 : n * v.seq) + (h / v.share) * v.head;
}

struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };

enum Form { OUT, OUT_TANGENT, SUM, SUM_TANGENT };   // an output (with the state's derivative by log g carried beside it); only what a segment adds

// DP: da and dc padded to 32, 64 or 128.  NW waves of CT column tiles each: NW * CT * 16 = DP.  VEC: every tensor is read and written
// 16 bytes (outputs: four values) at a time.
template <typename T, int DP, int NW, int CT, bool VEC, Form FORM> struct Sweep {
    typedef Mat<T> M;
    typedef typename M::Op Op;
    static constexpr bool TAN = FORM == OUT_TANGENT || FORM == SUM_TANGENT, ADD = FORM == SUM || FORM == SUM_TANGENT;
    static constexpr int NT = 64 * NW, LD = DP + M::VEC, TILES = DP / 16, KS = TILES / M::KT, RT = CHUNK / 16, KR = RT / M::KT;
    static constexpr int S2 = M::SPLIT ? (TAN ? 3 : 2) : 1, S3 = M::SPLIT ? 3 : 1;
    static constexpr int SCORES = RT * (RT + 1) / 2, MINE = (SCORES + NW - 1) / NW;             // score tiles; at most so many a wave
    static constexpr int PAIRS = M::KT == 2 ? RT / 2 * (RT / 2 + 1) : SCORES;                     // score operands: (it, kr), kr <= it / KT
    static constexpr int PIECE = CHUNK * LD;                                                      // one tensor's chunk in LDS
    static constexpr size_t BYTES = (ADD ? 2 : TAN ? 4 : 3) * PIECE * sizeof(T) + (ADD ? 0 : PAIRS * 64 * 16 * S2 * (TAN ? 2 : 1));
    static_assert(NW * CT == TILES, "every column tile has a wave");

    static __device__ __forceinline__ int pair(int it, int kr) { return M::KT == 2 ? (it >> 1) * ((it >> 1) + 1) + (it & 1) * ((it >> 1) + 1) + kr : it * (it + 1) / 2 + kr; }

    // four columns of a row, `left` of them there
    template <typename U> static __device__ __forceinline__ void put(U *base, uint32_t at, f32x4 v, int left) {
        typedef __attribute__((__vector_size__(4 * sizeof(U)))) U U4;
        U *to = (U *)((char *)base + (uint32_t)(at * sizeof(U)));
        if (VEC) {
            if (left > 0) *(U4 *)to = U4{(U)v[0], (U)v[1], (U)v[2], (U)v[3]};
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (r < left) to[r] = (U)v[r];
        }
    }

    static __device__ __forceinline__ void run(const Pass &P, char *lds) {
        T *const lb = (T *)lds, *const lc = lb + PIECE, *const la = lc + PIECE, *const le = la + PIECE;
        Op *const scores = (Op *)(lb + (TAN ? 4 : 3) * PIECE), *const slopes = scores + PAIRS * 64 * S2;      // [pair][term][lane]
        const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4, li = lane & 15;
        const int h = blockIdx.x % P.heads, slot = blockIdx.x / P.heads;
        const bool packed = P.offsets != nullptr;
        int n_seq, segment, lo, hi;
        slot_owner(P, slot, n_seq, segment);
        row_range(P.offsets, P.rows, n_seq, lo, hi);
        const int len = hi - lo, t0 = segment * P.seg_len;
        if (segment < 0 || (segment > 0 && t0 >= len)) {
            if (FORM == OUT_TANGENT && tid == 0) P.slope[blockIdx.x] = 0.0;
            return;
        }
        const bool last = len - t0 <= P.seg_len;
        if (ADD && last) return;
        const int t1 = last ? len : t0 + P.seg_len;
        // row t of the recurrence is row lo + t, or hi - 1 - t of a reversed pass; so a chunk of n begins at row low(t, n) of memory
        const auto low = [&](int t, int n) { return P.reverse ? hi - t - n : lo + t; };
        const T *pa = base_of<T>(P.a, packed, n_seq, h), *pb = base_of<T>(P.b, packed, n_seq, h), *pc = base_of<T>(P.c, packed, n_seq, h);
        const T *pe = FORM == OUT_TANGENT ? base_of<T>(P.e, packed, n_seq, h) : nullptr;
        Stage<T, DP, NT, VEC> sa, sb, sc, se;
        sb.init(P.b, tid);
        sc.init(P.c, tid);
        if (!ADD) sa.init(P.a, tid);
        if (FORM == OUT_TANGENT) se.init(P.e, tid);
        const auto fetch_as = [&](auto full, int t, int n) __attribute__((always_inline)) {
            constexpr bool FULL = decltype(full)::value;
            sb.template load<FULL>(pb, P.b, low(t, n), n, tid);
            if (!ADD) sa.template load<FULL>(pa, P.a, low(t, n), n, tid);
            sc.template load<FULL>(pc, P.c, low(t, n), n, tid);
            if (FORM == OUT_TANGENT) se.template load<FULL>(pe, P.e, low(t, n), n, tid);
        };
        const auto fetch = [&](int t) __attribute__((always_inline)) {
            if (t1 - t >= CHUNK) fetch_as(Yes(), t, CHUNK);
            else if (t < t1) fetch_as(No(), t, t1 - t);
        };
        fetch(t0);

        const float ld = P.log_decay[h], lg2 = ld * 1.44269504f;
        const int late = P.reverse ? 1 : 0;
        // g^64 as two floats: it multiplies the state once a chunk, and its own rounding would add up over a long memory
        const double whole_d = exp((double)ld * CHUNK);
        const float whole = (float)whole_d, whole_lo = isinf(whole) || whole == 0.0f ? 0.0f : (float)(whole_d - (double)whole);
        // weights: g^(i-j) us of this wave's score tiles; of row j of a full chunk in the state, g^(15 - its place in its tile) us, its tile's
        // factor beside it; g^(place of row i in its tile + 1), likewise
        float wa[MINE][4], wu[4];
        const float wo = power(lg2, li + 1 - late);
        float tiles[RT];                         // g^(16 k)
#pragma unroll
        for (int k = 0; k < RT; ++k) tiles[k] = power(lg2, 16 * k);
#pragma unroll
        for (int r = 0; r < 4; ++r) wu[r] = power(lg2, 15 - (g * 4 + r) + late) * P.upd_scale;
        int my_it[MINE], my_jt[MINE];
#pragma unroll
        for (int m = 0; m < MINE; ++m) {
            const int id = wave + NW * m;
            my_it[m] = id >= SCORES ? RT : id < 1 ? 0 : id < 3 ? 1 : id < 6 ? 2 : 3;
            my_jt[m] = id - my_it[m] * (my_it[m] + 1) / 2;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int apart = (my_it[m] - my_jt[m]) * 16 + li - (g * 4 + r);
                wa[m][r] = apart < 0 ? 0.0f : power(lg2, apart) * P.upd_scale;
            }
        }
        if (!ADD && M::KT == 2 && wave == 0) {      // the halves of operands above the diagonal
            const Op zero = {};
#pragma unroll
            for (int it = 0; it < RT; it += 2)
#pragma unroll
                for (int k = 0; k < S2; ++k) {
                    scores[(pair(it, it / 2) * S2 + k) * 64 + lane] = zero;
                    if (TAN) slopes[(pair(it, it / 2) * S2 + k) * 64 + lane] = zero;
                }
        }

        f32x4 S[TILES][CT], H[TAN ? TILES : 1][CT];
        const int64_t state_at = ((int64_t)n_seq * P.heads + h) * P.da * P.dc, seg_at = (int64_t)blockIdx.x * P.da * P.dc;
        const float *enter = ADD ? nullptr : segment > 0 ? P.seg + seg_at : P.state_in ? P.state_in + state_at : nullptr;
        const float *enter_tan = FORM == OUT_TANGENT && segment > 0 ? P.seg_tan + seg_at : nullptr;
#pragma unroll
        for (int mt = 0; mt < TILES; ++mt)
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                S[mt][ct] = f32x4{0, 0, 0, 0};
                if (TAN) H[mt][ct] = f32x4{0, 0, 0, 0};
            }
        if (enter) {
#pragma unroll
            for (int mt = 0; mt < TILES; ++mt)
#pragma unroll
                for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int i = mt * 16 + g * 4 + r, j = (wave * CT + ct) * 16 + li;
                        if (i < P.da && j < P.dc) {
                            S[mt][ct][r] = enter[i * P.st_a + j * P.st_c];
                            if (TAN && enter_tan) H[mt][ct][r] = enter_tan[i * P.st_a + j * P.st_c];
                        }
                    }
        }

        double slope = 0.0;
        const int64_t out_at = ((int64_t)(packed ? 0 : n_seq) * P.rows * P.heads + h) * P.dc;
        T *const out = (T *)P.out + out_at;
        float *const out_f32 = (float *)P.out + out_at;
        const auto chunk = [&](auto full, int t, int n_) __attribute__((always_inline)) {
            constexpr bool FULL = decltype(full)::value;
            const int n = FULL ? CHUNK : n_;
            sb.template store<FULL>(lb, pb, P.b, low(t, n), n, P.reverse, tid);
            sc.template store<FULL>(lc, pc, P.c, low(t, n), n, P.reverse, tid);
            if (!ADD) sa.template store<FULL>(la, pa, P.a, low(t, n), n, P.reverse, tid);
            if (FORM == OUT_TANGENT) se.template store<FULL>(le, pe, P.e, low(t, n), n, P.reverse, tid);
            __syncthreads();
            if (FULL) fetch(t + CHUNK);

            f32x4 o[RT][CT], x[TAN ? RT : 1][CT];
            if constexpr (!ADD) {
                // this wave's score tiles
#pragma unroll
                for (int m = 0; m < MINE; ++m) {
                    const int it = my_it[m], jt = my_jt[m];
                    if (it >= RT || (!FULL && it * 16 >= n)) continue;
                    f32x4 w = f32x4{0, 0, 0, 0}, wx;
#pragma unroll
                    for (int s = 0; s < KS; ++s) w = M::mma(M::row_op(lb, LD, jt * 16 + li, s, g), M::row_op(la, LD, it * 16 + li, s, g), w);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        w[r] *= wa[m][r];
                        if (TAN) wx[r] = w[r] * (float)((it - jt) * 16 + li - (g * 4 + r));
                    }
                    const int at = pair(it, jt / M::KT) * S2;
                    M::template keep<S2>(w, scores + at * 64 + lane, jt % M::KT);
                    if constexpr (TAN) M::template keep<S2>(wx, slopes + at * 64 + lane, jt % M::KT);
                }
                // F^T a
#pragma unroll
                for (int it = 0; it < RT; ++it)
#pragma unroll
                    for (int ct = 0; ct < CT; ++ct) {
                        o[it][ct] = f32x4{0, 0, 0, 0};
                        if (TAN) x[it][ct] = f32x4{0, 0, 0, 0};
                    }
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    Op f[CT][S2], ft[TAN ? CT : 1][S2];
#pragma unroll
                    for (int ct = 0; ct < CT; ++ct) {
                        f32x4 part[M::KT];
#pragma unroll
                        for (int k = 0; k < M::KT; ++k) part[k] = S[s * M::KT + k][ct];
                        M::template split<S2>(part, f[ct]);
                        if constexpr (TAN) {
#pragma unroll
                            for (int k = 0; k < M::KT; ++k) part[k] = H[s * M::KT + k][ct];
                            M::template split<S2>(part, ft[ct]);
                        }
                    }
#pragma unroll
                    for (int it = 0; it < RT; ++it) {
                        if (!FULL && it * 16 >= n) break;
                        const Op q = M::row_op(la, LD, it * 16 + li, s, g);
#pragma unroll
                        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                            for (int k = 0; k < S2; ++k) {
                                o[it][ct] = M::mma(f[ct][k], q, o[it][ct]);
                                if constexpr (TAN) x[it][ct] = M::mma(ft[ct][k], q, x[it][ct]);
                            }
                    }
                }
                __syncthreads();
            }

            Op vt[CT][KR];
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                for (int kr = 0; kr < KR; ++kr) vt[ct][kr] = M::col_op(lc, LD, wave * CT + ct, kr, g, li);

            if constexpr (!ADD) {
                // their weights, and the rows of this chunk
                float dot = 0.0f;
#pragma unroll
                for (int it = 0; it < RT; ++it) {
                    if (!FULL && it * 16 >= n) break;
                    const float into = wo * tiles[it];
#pragma unroll
                    for (int ct = 0; ct < CT; ++ct) {
                        if constexpr (TAN) x[it][ct] = (x[it][ct] + o[it][ct] * (float)(it * 16 + li + 1)) * into;
                        o[it][ct] = o[it][ct] * into;
                    }
#pragma unroll
                    for (int kr = 0; kr <= it / M::KT; ++kr)
#pragma unroll
                        for (int k = 0; k < S2; ++k) {
                            const int at = (pair(it, kr) * S2 + k) * 64 + lane;
                            const Op f = scores[at];
#pragma unroll
                            for (int ct = 0; ct < CT; ++ct) o[it][ct] = M::mma(vt[ct][kr], f, o[it][ct]);
                            if constexpr (TAN) {
                                const Op fx = slopes[at];
#pragma unroll
                                for (int ct = 0; ct < CT; ++ct) x[it][ct] = M::mma(vt[ct][kr], fx, x[it][ct]);
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
                        if (!P.out || (!FULL && i >= n)) continue;
                        const uint32_t by = (uint32_t)P.heads * P.dc, at = (P.reverse ? n - 1 - i : i) * by + col;
                        const f32x4 v = o[it][ct] * P.out_scale;
                        if (P.out_f32) put(out_f32 + (int64_t)low(t, n) * by, at, v, P.dc - col);
                        else put(out + (int64_t)low(t, n) * by, at, v, P.dc - col);
                    }
                }
                if (TAN) slope += (double)(dot * P.out_scale);
            }

            // F' = g^n F + sum_j g^(n-1-j) b_j c_j^T
            const float decay = FULL ? whole : power(lg2, n), decay_lo = FULL ? whole_lo : 0.0f;
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
                if (!FULL && kr * M::KT * 16 >= n) break;
                float w[M::KT][4];
                if (FULL) {
#pragma unroll
                    for (int k = 0; k < M::KT; ++k) {
                        const float tile = tiles[RT - 1 - (kr * M::KT + k)];
#pragma unroll
                        for (int r = 0; r < 4; ++r) w[k][r] = wu[r] * tile;
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < M::KT; ++k)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int j = (kr * M::KT + k) * 16 + g * 4 + r;
                            w[k][r] = j < n ? power(lg2, n - 1 - j + late) * P.upd_scale : 0.0f;
                        }
                }
                Op u[CT][S3], ux[TAN ? CT : 1][S3];
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) {
                    f32x4 y[M::KT], z[M::KT];
#pragma unroll
                    for (int k = 0; k < M::KT; ++k)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int j = (kr * M::KT + k) * 16 + g * 4 + r;
                            y[k][r] = M::elem(vt[ct][kr], k, r) * w[k][r];
                            if (TAN) z[k][r] = y[k][r] * (float)(n - 1 - j);
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
        };
        int t = t0;
        for (; t1 - t >= CHUNK; t += CHUNK) chunk(Yes(), t, CHUNK);
        if (t < t1) chunk(No(), t, t1 - t);

        float *leave = ADD ? P.seg + seg_at : last && P.state_out ? P.state_out + state_at : nullptr;
        float *leave_tan = FORM == SUM_TANGENT ? P.seg_tan + seg_at : nullptr;
        const float *grad = FORM == OUT_TANGENT && last && P.grad_state ? P.grad_state + state_at : nullptr;
        if (leave || grad) {
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
        }
        if constexpr (FORM == OUT_TANGENT) {
            double *red = (double *)lds;
            __syncthreads();
            red[tid] = slope;
            __syncthreads();
            for (int o = NT / 2; o > 0; o >>= 1) {
                if (tid < o) red[tid] += red[tid + o];
                __syncthreads();
            }
            if (tid == 0) P.slope[blockIdx.x] = red[0];
        }
    }
};

template <typename T, int DP, int NW, int CT, bool VEC, Form FORM, int WAVES> __global__ __launch_bounds__(64 * NW, WAVES) void td_decay_chunk_kernel(Pass P) {
    __shared__ __align__(16) char lds[Sweep<T, DP, NW, CT, VEC, FORM>::BYTES];
    Sweep<T, DP, NW, CT, VEC, FORM>::run(P, lds);
}

}  // namespace decay
