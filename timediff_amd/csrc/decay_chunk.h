// The chunked kernels of decay attention (decay_attn.hip has the formulas): a workgroup takes one sequence (or a segment of one) and
// head, 64 rows at a time, and keeps the state in registers between the chunks.  With i, j rows of a chunk of n, F the state
// entering it and X^T standing for a matrix with its columns in lanes,
//     out_i = os (g^(i+1) F^T a_i + sum_{j<=i} g^(i-j) (b_j . a_i) us c_j),       F' = g^n F + sum_j g^(n-1-j) us b_j c_j^T
// (reversed passes: rows counted from the chunk's end, out's exponent one less, F's terms' one more).  Everything is 16 x 16 matrix
// tiles, and the order of an operand's inner index is free as long as both operands share it, so that no product's result is ever
// moved between lanes:
//   * a wave owns 16 CT columns of c and of the state; the state's accumulators (rows = da in a lane's registers, lane = column) ARE
//     the operand of F^T a, and the scores' accumulators (rows j in registers, lane = row i) the operand of the sum over j: the waves
//     share out the ten score tiles on and below the diagonal and pass them on through LDS as operands, lane by lane;
//   * b and c are read from LDS with rows as the inner index by transposing loads (ds_read_b64_tr_b16).
// bfloat16: v_mfma_f32_16x16x32_bf16, and an operand that is not an input (scores, states, decayed rows that enter the state) is split into three
// bf16 terms, 2^-24 of it: a result is float32's, rounded once.  (Two terms for scores and states, 2^-17 of each, change one bfloat16 result in
// a few hundred.)  float32: v_mfma_f32_16x16x4_f32.
#pragma once
#include "common.h"

namespace decay {

constexpr int CHUNK = 64;

enum Kind { OUT, SUM, SUM_REVERSED, BACKWARD, BACKWARD_SLOPE };      // td_decay_out_kernel, td_decay_sum_kernel, td_decay_backward_kernel

struct View {                 // rows of one tensor; head h of the recurrence reads head h / share
    const void *p;
    int64_t seq, row, head;
    int share, d;
    int pairs;                // bfloat16: two neighbours can be read at once
};

struct Pass {
    View a, b, c, e;          // ascending: out from (a, b, c), e: what the slope of out is dotted with.  Descending: out from (a, b, c), out2 from (e, c, b)
    const float *log_decay;
    const int32_t *offsets;   // packed: n_seq + 1, else NULL
    const float *state_in;    // (n_seq, heads, ..): element (i, j) of (da, dc) at i * st_a + j * st_c, NULL: zeros
    float *state_out;         // NULL: not wanted
    float *seg;               // (slots, heads, ..) as state_in: the state entering each segment; SUM: what each one adds
    double *slope;            // one sum for each (slot, head)
    int64_t st_a, st_c;
    void *out, *out2;         // (rows, heads, dc), (rows, heads, da), float32 (out_f32, out2_f32) or the tensors' type; NULL: not wanted
    int out_f32, out2_f32;
    int n_seq, rows, heads, da, dc;
    int seg_len, segs, slots; // rows of a segment (a multiple of CHUNK), segments of a dense sequence (1: seg_len covers all), slots in all
    int first;                // workgroup 0's place among all of them (launch_parts)
    float out_scale, upd_scale;
};

// HIP launches fewer than 2^32 threads at once: `groups` workgroups in as many launches as that takes
template <typename L> void launch_parts(Pass P, int64_t groups, int threads, L launch) {
    const int64_t most = 0xFFFFFFFFll / threads;
    for (int64_t at = 0; at < groups; at += most) {
        P.first = (int)at;
        launch(P, dim3((unsigned)(groups - at < most ? groups - at : most)));
    }
}

// What a launcher takes.  Backward: p ascending, r descending, `groups` workgroups that share out the slots and heads
struct Work {
    Pass p, r;
    float *chunk_states;
    int groups, ascending, descending;
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

// Packed sequence n owns the places from lo(n) / size + n on, for segments (size = seg_len) as for chunks: a sequence of any length has as
// many as it needs (one at least), no two share one, and there are rows / size + n_seq in all, whatever the lengths are.
__device__ __forceinline__ int first_place(const Pass &P, int n, int size) { return min(max(P.offsets[n], 0), P.rows) / size + n; }

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
        if (first_place(P, mid, P.seg_len) <= slot) lo = mid;
        else hi = mid - 1;
    }
    n = lo;
    segment = slot - first_place(P, lo, P.seg_len);
}

// log2 g as two floats.  One float alone, multiplied by e, leaves 2^-24 |log2 g^e| twice in the exponent: a weight of 2^-50 would be off by 40
// roundings.  Finite (g = 0 is 2^-1e30), so that e = 0 gives 1.
struct Log2 {
    float hi, lo;
    static __device__ __forceinline__ Log2 of(float log_g) {
        log_g = log_g < -1e30f ? -1e30f : log_g > 1e30f ? 1e30f : log_g;
        const float x = log_g * 1.44269502f;                       // log2(e) = 1.44269502162933 + 1.92596299e-8
        return Log2{x, __builtin_fmaf(log_g, 1.92596299e-8f, __builtin_fmaf(log_g, 1.44269502f, -x))};
    }
};

// g^e for a whole number e: 2^x by the hardware (one unit in the last place), times 1 and what x leaves out, to first order (half a unit at
// most while 2^x is neither 0 nor infinite; the bound keeps those two what they are).  No selection: the compiler makes branches of them, and between
// matrix instructions a branch is a place where it has left out waits.
__device__ __forceinline__ float power(Log2 lg2, int e) {
    const float n = (float)e, x = lg2.hi * n, rest = __builtin_fmaf(lg2.lo, n, __builtin_fmaf(lg2.hi, n, -x));
    return __builtin_amdgcn_exp2f(x) * fmaxf(__builtin_fmaf(rest, 0.693147181f, 1.0f), 0.5f);
}

// g^e as two floats: it multiplies a state again and again, and its own rounding would add up over a long memory
struct Factor { float hi, lo; };
__device__ __forceinline__ Factor factor(float log_g, int e) {
    const double x = e == 0 ? 1.0 : exp((double)log_g * e);
    const float hi = (float)x;
    return Factor{hi, isinf(hi) || hi == 0.0f ? 0.0f : (float)(x - (double)hi)};
}
__device__ __forceinline__ float times(Factor f, float x) { return __builtin_fmaf(f.hi, x, f.lo * x); }

template <typename T> struct Mat;
template <> struct Mat<__bf16> {
    typedef bf16x8 Op;
    static constexpr int KT = 2;        // tiles of 16 that an operand spans
    static constexpr int VEC = 8;       // elements of 16 bytes
    static constexpr bool SPLIT = true;
    static __device__ __forceinline__ f32x4 mma(Op a, Op b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    static constexpr int pitch(int d) { return d; }          // elements between rows in LDS
    static __device__ __forceinline__ Op row_op(const __bf16 *t, int d, int row, int ks, int g) { return *(const Op *)(t + lds_at(d, row, ks * 4 + g)); }
    static __device__ __forceinline__ Op col_op(const __bf16 *t, int d, int tile, int kr, int g, int li) {
        typedef __attribute__((__vector_size__(4 * sizeof(short)))) short s16x4;
        typedef __attribute__((address_space(3))) s16x4 *lds;
        const int row = kr * 32 + g * 4 + (li >> 2);
        const __bf16 *p = t + lds_at(d, row, (tile >> 1) * 4 + (li & 3)) + (tile & 1) * 4;
        union { s16x4 s[2]; Op o; } x;
        x.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(void *)p);
        x.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(void *)(p + 16 * d));
        return x.o;
    }
    // A row in LDS: of each 32 columns, 16 bytes for each group g with its four of the first 16 and its four of the second (the order of an
    // operand's inner index, so that one 16-byte load is an operand); no padding, a row's 16-byte pieces change places with
    // bits of the row's number, so that eight rows' same piece and four rows' four neighbouring pieces both lie on different banks.
    static __device__ __forceinline__ int lds_at(int d, int row, int piece) {
        const int turn = d == 64 ? (row & 2) << 1 | (row & 4) >> 1 | (row & 1) : d > 64 ? (row & 3) << 2 | (row & 4) >> 2 : (row & 4) >> 2;
        return row * d + (piece ^ turn) * 8;
    }
    // four columns from 4 * four on
    static __device__ __forceinline__ int four_at(int d, int row, int four) { return lds_at(d, row, (four >> 3) * 4 + (four & 3)) + ((four >> 2) & 1) * 4; }
    // two values to bf16 (one instruction); what is left of them behind
    static __device__ __forceinline__ uint32_t term(float &a, float &b, bool last) {
        typedef __attribute__((ext_vector_type(2))) float f32x2;
        typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
        const uint32_t bits = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
        if (!last) {
            a -= __uint_as_float(bits << 16);
            b -= __uint_as_float(bits & 0xFFFF0000u);
        }
        return bits;
    }
    // the operand whose elements are x[tile][register]
    template <int N> static __device__ __forceinline__ void split(const f32x4 *x, Op *p) {
        union { uint32_t u[4]; Op o; } y[N];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float a = x[j >> 1][2 * j & 3], b = x[j >> 1][(2 * j & 3) + 1];
#pragma unroll
            for (int k = 0; k < N; ++k) y[k].u[j] = term(a, b, k == N - 1);
        }
#pragma unroll
        for (int k = 0; k < N; ++k) p[k] = y[k].o;
    }
    // one tile's terms into its half of the operands at to, to + 64, ..
    template <int N> static __device__ __forceinline__ void keep(f32x4 x, Op *to, int half) {
        float a = x[0], b = x[1], c = x[2], d = x[3];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const uint32_t low = term(a, b, k == N - 1), high = term(c, d, k == N - 1);
            *((uint2 *)(to + 64 * k) + half) = uint2{low, high};
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
    static constexpr int pitch(int d) { return d + 4; }      // rows in LDS: 16 bytes between them
    static __device__ __forceinline__ Op row_op(const float *t, int d, int row, int ks, int g) { return *(const Op *)(t + row * pitch(d) + ks * 16 + g * 4); }
    static __device__ __forceinline__ Op col_op(const float *t, int d, int tile, int kr, int g, int li) {
        const float *p = t + (kr * 16 + g * 4) * pitch(d) + tile * 16 + li;
        return Op{p[0], p[pitch(d)], p[2 * pitch(d)], p[3 * pitch(d)]};
    }
    static __device__ __forceinline__ int four_at(int d, int row, int four) { return row * pitch(d) + four * 4; }
    template <int N> static __device__ __forceinline__ void split(const f32x4 *x, Op *p) { p[0] = x[0]; }
    template <int N> static __device__ __forceinline__ void keep(f32x4 x, Op *to, int) { *to = x; }
    static __device__ __forceinline__ float elem(Op o, int, int r) { return o[r]; }
};

// A chunk's rows: a whole chunk, or the last rows of a sequence, of which tiles of 16 there are at most LIVE.  (How many tiles a product covers is
// a constant in each form: a branch on it would stand between a matrix instruction and the readers of its result.)
template <int LIVE_, bool FULL_> struct Rows {
    static constexpr int LIVE = LIVE_;
    static constexpr bool FULL = FULL_;
};
typedef Rows<CHUNK / 16, true> Whole;
typedef Rows<CHUNK / 16, false> Most;
typedef Rows<CHUNK / 32, false> Half;

// One chunk's rows of one tensor on their way from memory to LDS.  Memory is read in the order of its rows (n of them from `low` on), a
// reversed pass turns them round in LDS.  The loads go into registers while the chunk before is computed (unless there are too many of them:
// 64 bytes of each tensor a thread; 4 bytes at a time in workgroups of 512 threads, whose registers four tensors would fill, 32: 101 x 101 float32,
// 16 sequences of 1024 rows, 8 heads: 852 us backward, 1032 with 64.  Rectangles, two of whose tensors take 32 anyway, would gain with 64:
// 41 x 101 458 and 381, 101 x 41 589 and 581).
// WIDE: 16 bytes each, at 32-bit offsets from the chunk's first row; else (odd sizes, strides or addresses) 4 bytes each.  They are never
// skipped, so that their registers have one writer: a lane without a row or a column of its own reads its neighbours', and
// nothing of that is stored.
template <typename T, int D, int NT, bool WIDE, bool REV> struct Stage {
    static constexpr int BYTES = WIDE ? 16 : 4, PER = BYTES / sizeof(T), PIECES = D / PER, N = CHUNK * PIECES / NT;
    static constexpr bool AHEAD = N * BYTES <= (WIDE || NT < 512 ? 64 : 32);
    static_assert(NT % PIECES == 0, "a thread's pieces share their columns");
    struct Wide { uint4 x; };
    struct Narrow { uint32_t x; };
    template <bool W, typename A, typename B> struct Pick { typedef A Type; };
    template <typename A, typename B> struct Pick<false, A, B> { typedef B Type; };
    typedef decltype(Pick<WIDE, Wide, Narrow>::Type::x) Piece;
    Piece r[AHEAD ? N : 1];
    // the columns behind the last are zeros from here on
    static __device__ __forceinline__ void init(T *lds, const View &v, int tid) {
        if (v.d < D)
            for (int i = tid; i < CHUNK * Mat<T>::pitch(D); i += NT) lds[i] = (T)0.0f;
    }
    static __device__ __forceinline__ Piece piece(const char *chunk, const View &v, int c, int n, int tid) {
        const int row = min(tid / PIECES + c * (NT / PIECES), n - 1), own = tid % PIECES * PER;
        if constexpr (WIDE) {
            const int col = min(own, v.d - PER);
            return *(const uint4 *)(chunk + (uint32_t)(__umul24(row, (uint32_t)v.row * sizeof(T)) + col * sizeof(T)));
        } else if constexpr (sizeof(T) == 4) {
            return *(const uint32_t *)(chunk + (row * v.row + min(own, v.d - 1)) * (int64_t)sizeof(T));
        } else {
            const uint16_t *p = (const uint16_t *)chunk + row * v.row;
            if (v.pairs) return *(const uint32_t *)(p + min(own, v.d - 2));
            return (uint32_t)p[min(own, v.d - 1)] | (own + 1 < v.d ? (uint32_t)p[min(own + 1, v.d - 1)] << 16 : 0u);
        }
    }
    // n >= 1
    __device__ __forceinline__ void load(const T *base, const View &v, int low, int n, int tid) {
        if (!AHEAD) return;
        const char *chunk = (const char *)(base + (int64_t)low * v.row);
#pragma unroll
        for (int c = 0; c < N; ++c) r[c] = piece(chunk, v, c, n, tid);
    }
    // the tiles of rows that R has
    template <typename R> __device__ __forceinline__ void store(T *lds, const T *base, const View &v, int low, int n, int tid) const {
        constexpr bool FULL = R::FULL;
        constexpr int AT_ONCE = NT / PIECES, LAST = (R::LIVE * 16 + AT_ONCE - 1) / AT_ONCE;
        if (tid % PIECES * PER >= v.d) return;
        const char *chunk = (const char *)(base + (int64_t)low * v.row);
#pragma unroll
        for (int c = 0; c < LAST; ++c) {
            const int row = tid / PIECES + c * (NT / PIECES), at = tid % PIECES, to = REV && (FULL || row < n) ? (FULL ? CHUNK : n) - 1 - row : row;
            Piece x = AHEAD ? r[AHEAD ? c : 0] : piece(chunk, v, c, FULL ? CHUNK : n, tid);
            if (!FULL && row >= n) x = Piece{};
            if constexpr (!WIDE) {
                *(uint32_t *)(lds + Mat<T>::four_at(D, to, at * PER >> 2) + (at * PER & 3)) = x;
            } else if constexpr (PER == 8) {
                *(uint2 *)(lds + Mat<T>::four_at(D, to, 2 * at)) = uint2{x.x, x.y};
                *(uint2 *)(lds + Mat<T>::four_at(D, to, 2 * at + 1)) = uint2{x.z, x.w};
            } else {
                *(uint4 *)(lds + Mat<T>::four_at(D, to, at)) = x;
            }
        }
    }
};

// The next chunk of a pass, for the loads ahead: its first row and how many it has (1 where there is none: a row that is there)
struct Next { int t, n; };

template <typename T> __device__ __forceinline__ const T *base_of(const View &v, bool packed, int n, int h) {
    return (const T *)v.p + (packed ? 0 : n * v.seq) + (h / v.share) * v.head;
}

// The thread's number as if read anew: what is computed from it (addresses in LDS and in memory, places in a tile) is computed again where it
// is used.  Kept from chunk to chunk, as the compiler would, it fills the registers twice over.
__device__ __forceinline__ int here(int tid) {
    asm volatile("" : "+v"(tid));
    return tid;
}

// A kernel's argument of type A at byte `at` of the argument list, read anew from memory where it is used: kept in scalar registers, the
// two passes' arguments would be spilled lane by lane.
template <typename A> __device__ __forceinline__ const A &argument(int at) {
    typedef const __attribute__((address_space(4))) char *Args;
    Args p = (Args)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const A *)(const char *)(p + at);
}

// Loads of what comes behind stay behind: the registers of two steps at once do not fit
__device__ __forceinline__ void phase() { __builtin_amdgcn_sched_barrier(0); }

// Waits until the matrix instructions before it have written their results.  It stands wherever a branch (a loop's end, a store of some
// lanes) comes between a matrix instruction and the first reader of its result: the compiler places the waits that the hardware
// needs itself, but on some paths through a branch it has left them out (results of v_mfma_f32_16x16x4_f32 were read 1 instruction behind it
// instead of 10).
__device__ __forceinline__ void settle() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 15");
    __builtin_amdgcn_sched_barrier(0);
}

template <bool V> struct Flag { static constexpr bool value = V; };

// Which segment of which sequence a workgroup has
struct Place {
    int n_seq, segment, lo, t0, t1;      // rows lo + t0 .. lo + t1 - 1
    bool last;
    __device__ __forceinline__ bool find(const Pass &P, int slot) {
        int hi;
        slot_owner(P, slot, n_seq, segment);
        row_range(P.offsets, P.rows, n_seq, lo, hi);
        if (segment < 0 || (segment > 0 && (int64_t)segment * P.seg_len >= hi - lo)) return false;
        t0 = segment * P.seg_len;
        last = hi - lo - t0 <= P.seg_len;
        t1 = last ? hi - lo : t0 + P.seg_len;
        return true;
    }
};

// The weights of a head that every chunk uses
template <int NW> struct Weights {
    static constexpr int RT = CHUNK / 16, SCORES = RT * (RT + 1) / 2, MINE = (SCORES + NW - 1) / NW;   // score tiles; at most so many a wave
    Log2 lg2;
    float wo, wu[4], wa[MINE][4], tiles[RT];
    int it[MINE], jt[MINE];
    Factor whole;
    // late: 1 in reversed passes
    __device__ __forceinline__ void init(float log_g, float scale, int late, int wave, int g, int li) {
        lg2 = Log2::of(log_g);
        whole = factor(log_g, CHUNK);
        wo = power(lg2, li + 1 - late);                                             // of row i: g^(its place in its tile + 1), times
#pragma unroll
        for (int k = 0; k < RT; ++k) tiles[k] = power(lg2, 16 * k);                 // g^(16 tiles before its own)
#pragma unroll
        for (int r = 0; r < 4; ++r) wu[r] = power(lg2, 15 - (g * 4 + r) + late) * scale;   // of row j in the state, likewise from the chunk's end
#pragma unroll
        for (int m = 0; m < MINE; ++m) {                                            // of this wave's score tiles: g^(i-j)
            const int id = wave + NW * m;
            it[m] = id >= SCORES ? RT : id < 1 ? 0 : id < 3 ? 1 : id < 6 ? 2 : 3;
            jt[m] = id - it[m] * (it[m] + 1) / 2;
#pragma unroll
            for (int r = 0; r < 4; ++r) wa[m][r] = apart(m, r, g, li) < 0 ? 0.0f : power(lg2, apart(m, r, g, li)) * scale;
        }
    }
    __device__ __forceinline__ int apart(int m, int r, int g, int li) const { return (it[m] - jt[m]) * 16 + li - (g * 4 + r); }
    // Whether a pair of rows counts: not those above the diagonal or behind the n-th row, where a product of finite values may have overflowed
    template <typename R> __device__ __forceinline__ bool pair(int m, int r, int n, int g, int li) const {
        return apart(m, r, g, li) >= 0 && (R::FULL || it[m] * 16 + li < n);
    }
    template <typename R> __device__ __forceinline__ float weigh(float s, int m, int r, int n, int g, int li) const { return pair<R>(m, r, n, g, li) ? s * wa[m][r] : 0.0f; }
};

// Which of a chunk's four row tiles a wave's outputs have.  NI = 4: all of them.  NI = 2: two teams of waves hold the same state, team 0 has the
// outputs of tiles 0 and 3, team 1 those of 1 and 2: as many products with scores (and in `most` of two tiles, as many tiles) for each.
template <int NI> struct Tiles {
    int team;
    float factor[NI];            // g^(16 tile)
    __device__ __forceinline__ void init(Log2 lg2, int team_) {
        team = team_;
#pragma unroll
        for (int j = 0; j < NI; ++j) factor[j] = power(lg2, 16 * at(j));
    }
    __device__ __forceinline__ int at(int j) const { return NI == 4 ? j : j == 0 ? team : 3 - team; }
    static constexpr bool live(int j, int most) { return NI == 4 ? j < most : j == 0 || most > 2; }
};

// One product stream: the state M (DA x DC) and what a chunk does with it.  TA x CT tiles of the state a wave.
template <typename T, int DA, int DC, int NW, bool VEC, int NI = 4> struct Stream {
    typedef Mat<T> M;
    typedef typename M::Op Op;
    static constexpr int PER = 2 / M::KT;                // operands of 32 rows
    static constexpr int LA = DA, LC = DC, PA = M::pitch(DA), PC = M::pitch(DC), TA = DA / 16, CT = DC / 16 / NW, KS = TA / M::KT, RT = CHUNK / 16, KR = RT / M::KT;
    static constexpr int TERMS = M::SPLIT ? 3 : 1;      // of scores, of decayed rows and of the state
    static constexpr int PAIRS = M::KT == 2 ? RT / 2 * (RT / 2 + 1) : RT * (RT + 1) / 2;               // score operands: (it, kr), kr <= it / KT
    static_assert(CT * NW * 16 == DC && CT > 0, "every column tile has a wave");
    f32x4 S[TA][CT], o[NI][CT];
    Op vt[CT][KR];
    Tiles<NI> tiles;

    static __device__ __forceinline__ int pair(int it, int kr) { return M::KT == 2 ? (it >> 1) * ((it >> 1) + 1) + (it & 1) * ((it >> 1) + 1) + kr : it * (it + 1) / 2 + kr; }
    // score operands of row tile j; with two teams as many for both, a tile of zeros where a team's own tile has one less
    static constexpr int operands(int j) { return NI == 4 ? j / M::KT + 1 : M::KT == 2 ? j + 1 : 2 * j + 2; }

    // the halves of score operands above the diagonal
    static __device__ __forceinline__ void clear_scores(Op *scores, int lane) {
        const Op zero = {};
        if (M::KT == 2)
#pragma unroll
            for (int it = 0; it < RT; it += 2)
#pragma unroll
                for (int k = 0; k < TERMS; ++k) scores[(pair(it, it / 2) * TERMS + k) * 64 + lane] = zero;
    }
    // (b_j . a_i) of tile (it, jt)
    static __device__ __forceinline__ f32x4 score(const T *la, const T *lb, int it, int jt, int g, int li) {
        f32x4 w = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < KS; ++s) w = M::mma(M::row_op(lb, LA, jt * 16 + li, s, g), M::row_op(la, LA, it * 16 + li, s, g), w);
        return w;
    }
    static __device__ __forceinline__ void keep(f32x4 w, Op *scores, int it, int jt, int lane) {
        M::template keep<TERMS>(w, scores + pair(it, jt / M::KT) * TERMS * 64 + lane, jt % M::KT);
    }
    __device__ __forceinline__ void enter(const float *from, int64_t st_a, int64_t st_c, int da, int dc, int wave, int g, int li) {
#pragma unroll
        for (int mt = 0; mt < TA; ++mt)
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) S[mt][ct] = f32x4{0, 0, 0, 0};
        if (!from) return;
#pragma unroll
        for (int mt = 0; mt < TA; ++mt)
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = mt * 16 + g * 4 + r, j = (wave * CT + ct) * 16 + li;
                    if (i < da && j < dc) S[mt][ct][r] = from[i * st_a + j * st_c];
                }
    }
    __device__ __forceinline__ void leave(float *to, int64_t st_a, int64_t st_c, int da, int dc, int wave, int g, int li) const {
        if (!to) return;
#pragma unroll
        for (int mt = 0; mt < TA; ++mt)
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = mt * 16 + g * 4 + r, j = (wave * CT + ct) * 16 + li;
                    if (i < da && j < dc) to[i * st_a + j * st_c] = S[mt][ct][r];
                }
    }
    // o = g^(i+1) F^T a (rows behind the n-th have no weight: g^(i+1) of a growing state may be infinite there)
    template <typename R, typename W> __device__ __forceinline__ void from_state(const T *la, int n, const W &w, int g, int li) {
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) o[j][ct] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            Op f[CT][TERMS];
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                f32x4 part[M::KT];
#pragma unroll
                for (int k = 0; k < M::KT; ++k) part[k] = S[s * M::KT + k][ct];
                M::template split<TERMS>(part, f[ct]);
            }
#pragma unroll
            for (int j = 0; j < NI; ++j) {
                if (!tiles.live(j, R::LIVE)) continue;
                const Op q = M::row_op(la, LA, tiles.at(j) * 16 + li, s, g);
#pragma unroll
                for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                    for (int k = 0; k < TERMS; ++k) o[j][ct] = M::mma(f[ct][k], q, o[j][ct]);
            }
        }
#pragma unroll
        for (int j = 0; j < NI; ++j) {
            const float weight = R::FULL || tiles.at(j) * 16 + li < n ? w.wo * tiles.factor[j] : 0.0f;
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) o[j][ct] = o[j][ct] * weight;
        }
    }
    // sum of (first + i) o_i . e_i over this lane's entries
    template <typename R> __device__ __forceinline__ float dot(const T *le, int first, int wave, int g, int li) const {
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < NI; ++j) {
            if (!tiles.live(j, R::LIVE)) continue;
            const int i = tiles.at(j) * 16 + li;
            float part = 0.0f;
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                const T *e = le + M::four_at(LC, i, (wave * CT + ct) * 4 + g);
#pragma unroll
                for (int r = 0; r < 4; ++r) part += o[j][ct][r] * (float)e[r];
            }
            sum += (float)(first + i) * part;
        }
        return sum;
    }
    template <typename R> __device__ __forceinline__ void columns(const T *lc, int wave, int g, int li) {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int kr = 0; kr < (R::LIVE + M::KT - 1) / M::KT; ++kr) vt[ct][kr] = M::col_op(lc, LC, wave * CT + ct, kr, g, li);
    }
    // o += the rows of this chunk; rows of o to memory
    template <typename R, bool REV> __device__ __forceinline__ void from_rows(const Op *scores, int n, float scale, void *out, int out_f32, int64_t row0, int heads, int h, int dc,
                                                                             int wave, int lane) {
        if (!out) return;
        const int g = lane >> 4, li = lane & 15;
        const uint32_t by = (uint32_t)heads * dc;
        const int64_t first = row0 * by + (int64_t)h * dc;
#pragma unroll
        for (int j = 0; j < NI; ++j) {
            if (!tiles.live(j, R::LIVE)) continue;
#pragma unroll
            for (int kr = 0; kr < operands(j); ++kr)
#pragma unroll
                for (int k = 0; k < TERMS; ++k) {
                    Op f = scores[(pair(tiles.at(j), kr) * TERMS + k) * 64 + lane];
                    if (NI == 2 && M::KT == 1) f = kr <= tiles.at(j) ? f : Op{};
#pragma unroll
                    for (int ct = 0; ct < CT; ++ct) o[j][ct] = M::mma(vt[ct][kr], f, o[j][ct]);
                }
        }
        settle();                 // the lanes without a row branch past the readers
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) o[j][ct] = o[j][ct] * scale;
#pragma unroll
        for (int j = 0; j < NI; ++j) {
            const int i = tiles.at(j) * 16 + li;
            if (!tiles.live(j, R::LIVE) || (!R::FULL && i >= n)) continue;
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                const int col = (wave * CT + ct) * 16 + g * 4;
                const uint32_t at = (uint32_t)(REV ? n - 1 - i : i) * by + col;
                if (out_f32) put((float *)out + first, at, o[j][ct], dc - col);
                else put((T *)out + first, at, o[j][ct], dc - col);
            }
        }
    }
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
    // F' = g^n F + sum_j g^(n-1-j+late) us b_j c_j^T.  float32: 32 rows are summed before they enter the state, whose roundings stay, chunk after chunk
    // (added by fours, results of 271 rows were off by 2.5e-7 of their norm and are by 1.9e-7, states of some thousand rows by 5e-7 and 1.5e-7).
    template <typename R, typename W> __device__ __forceinline__ void advance(const T *lb, int n, const W &w, float scale, int late, int g, int li) {
        const Factor f = R::FULL ? w.whole : Factor{power(w.lg2, n), 0.0f};
        if (M::SPLIT)
#pragma unroll
            for (int mt = 0; mt < TA; ++mt)
#pragma unroll
                for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                    for (int r = 0; r < 4; ++r) S[mt][ct][r] = times(f, S[mt][ct][r]);
#pragma unroll
        for (int half = 0; half < (R::LIVE + 1) / 2; ++half) {
            Op u[CT][PER][TERMS];
#pragma unroll
            for (int p = 0; p < PER; ++p) {
                float wr[M::KT][4];
#pragma unroll
                for (int k = 0; k < M::KT; ++k)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int tile = half * 2 + p * M::KT + k, j = tile * 16 + g * 4 + r;
                        wr[k][r] = R::FULL ? w.wu[r] * w.tiles[RT - 1 - tile] : j < n ? power(w.lg2, n - 1 - j + late) * scale : 0.0f;
                    }
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) {
                    f32x4 y[M::KT];
#pragma unroll
                    for (int k = 0; k < M::KT; ++k)
#pragma unroll
                        for (int r = 0; r < 4; ++r) y[k][r] = M::elem(vt[ct][half * PER + p], k, r) * wr[k][r];
                    M::template split<TERMS>(y, u[ct][p]);
                }
            }
#pragma unroll
            for (int mt = 0; mt < TA; ++mt) {
                f32x4 add[CT];
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) add[ct] = M::SPLIT ? S[mt][ct] : f32x4{0, 0, 0, 0};
#pragma unroll
                for (int p = 0; p < PER; ++p) {
                    const Op b = M::col_op(lb, LA, mt, half * PER + p, g, li);
#pragma unroll
                    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                        for (int k = 0; k < TERMS; ++k) add[ct] = M::mma(b, u[ct][p][k], add[ct]);
                }
#pragma unroll
                for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float x = S[mt][ct][r];
                        S[mt][ct][r] = M::SPLIT ? add[ct][r] : half == 0 ? __builtin_fmaf(f.hi, x, __builtin_fmaf(f.lo, x, add[ct][r])) : x + add[ct][r];
                    }
            }
        }
        settle();
        settle();
    }
};

// Rows of no sequence: zeros in head h's columns, shared out over the slots
template <typename U> __device__ __forceinline__ void clear_rows(const Pass &P, U *out, int dc, int slot, int h, int tid, int nt) {
    const int lo = min(max(P.offsets[0], 0), P.rows), hi = min(max(P.offsets[P.n_seq], lo), P.rows);
    for (int64_t i = slot; i < lo + (P.rows - hi); i += P.slots)
        for (int c = tid; c < dc; c += nt) out[((i < lo ? i : hi + (i - lo)) * P.heads + h) * dc + c] = (U)0.0f;
}
template <typename T> __device__ __forceinline__ void clear_rows_of(const Pass &P, void *out, int f32, int dc, int slot, int h, int tid, int nt) {
    if (!out) return;
    if (f32) clear_rows(P, (float *)out, dc, slot, h, tid, nt);
    else clear_rows(P, (T *)out, dc, slot, h, tid, nt);
}

// The sum of a workgroup's values, in a fixed order: inside the waves, then wave by wave
template <int NT> __device__ __forceinline__ void workgroup_sum(double x, double *red, double *to, int tid) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
    __syncthreads();
    if ((tid & 63) == 0) red[tid >> 6] = x;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < NT / 64; ++w) x += red[w];
        *to = x;
    }
}

// What a segment adds to the state
template <typename T, int DA, int DC, int NW, bool VEC, bool REV, int WAVES> __global__ __launch_bounds__(64 * NW, WAVES) void td_decay_sum_kernel(Pass P) {
    typedef Stream<T, DA, DC, NW, VEC> X;
    constexpr int NT = 64 * NW;
    __shared__ __align__(16) T lb[CHUNK * X::PA];
    __shared__ __align__(16) T lc[CHUNK * X::PC];
    const int tid_ = here(threadIdx.x), tid = tid_, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = (tid & 63) >> 4, li = tid & 15;
    const int item = P.first + blockIdx.x, h = item % P.heads, slot = item / P.heads;
    Place at;
    if (!at.find(P, slot) || (REV ? at.segment == 0 : at.last)) return;      // nothing enters a segment from these
    const T *pb = base_of<T>(P.b, P.offsets, at.n_seq, h) + (int64_t)at.lo * P.b.row, *pc = base_of<T>(P.c, P.offsets, at.n_seq, h) + (int64_t)at.lo * P.c.row;
    Stage<T, DA, NT, VEC, REV> sb;
    Stage<T, DC, NT, VEC, REV> sc;
    sb.init(lb, P.b, tid);
    sc.init(lc, P.c, tid);
    const auto fetch = [&](Next next, int tid) __attribute__((always_inline)) {
        sb.load(pb, P.b, next.t, next.n, tid);
        sc.load(pc, P.c, next.t, next.n, tid);
    };
    const int whole = (at.t1 - at.t0) / CHUNK, tail = (at.t1 - at.t0) % CHUNK;
    fetch(REV && tail ? Next{at.t1 - tail, tail} : Next{REV ? at.t1 - CHUNK : at.t0, CHUNK}, tid);
    __syncthreads();
    Weights<NW> w;
    w.init(P.log_decay[h], P.upd_scale, REV, wave, g, li);
    X x;
    x.enter(nullptr, 0, 0, 0, 0, wave, g, li);
    const auto chunk = [&](auto rows, int t, int n, Next next) __attribute__((always_inline)) {
        typedef decltype(rows) R;
        constexpr bool FULL = R::FULL;
        const int tid = here(tid_), lane = tid & 63, g = lane >> 4, li = lane & 15;
        sb.template store<R>(lb, pb, P.b, t, n, tid);
        sc.template store<R>(lc, pc, P.c, t, n, tid);
        __syncthreads();
        fetch(next, tid);
        x.template columns<R>(lc, wave, g, li);
        x.template advance<R>(lb, n, w, P.upd_scale, REV, g, li);
        __syncthreads();
    };
    const Next before = whole ? Next{at.t1 - tail - CHUNK, CHUNK} : Next{at.t0, 1};
    if (REV && tail > CHUNK / 2) chunk(Most(), at.t1 - tail, tail, before);
    else if (REV && tail) chunk(Half(), at.t1 - tail, tail, before);
    for (int c = 0; c < whole; ++c) {        // (a segment that is not the last has no tail)
        const int t = REV ? at.t0 + (whole - 1 - c) * CHUNK : at.t0 + c * CHUNK;
        chunk(Whole(), t, CHUNK, c + 1 < whole ? Next{REV ? t - CHUNK : t + CHUNK, CHUNK} : Next{t, 1});
    }
    x.leave(P.seg + (int64_t)item * P.da * P.dc, P.st_a, P.st_c, P.da, P.dc, wave, g, li);
}

// out from (a, b, c), rows ascending.  SLOPE: the part of the derivative by log g that rows owe to the states entering their chunks, dotted with
// e, and those states for the pass over the other gradients.
template <typename T, int DA, int DC, int NW, bool SLOPE> struct OutLds {
    typedef Stream<T, DA, DC, NW, true> X;
    T a[CHUNK * X::PA], b[CHUNK * X::PA], c[CHUNK * X::PC], e[SLOPE ? CHUNK * X::PC : 8];
    typename X::Op scores[X::PAIRS * X::TERMS * 64];
};
template <typename T, int DA, int DC, int NW, int TEAMS, bool VEC, bool SLOPE>
__device__ __forceinline__ void out_sweep(const Pass &P, int item, OutLds<T, DA, DC, NW, SLOPE> &lds, float *chunk_states) {
    typedef Stream<T, DA, DC, NW, VEC, 4 / TEAMS> X;
    typedef typename X::Op Op;
    constexpr int NT = 64 * NW * TEAMS;
    T *const la = lds.a, *const lb = lds.b, *const lc = lds.c, *const le = lds.e;
    Op *const scores = lds.scores;
    const int tid_ = here(threadIdx.x), tid = tid_, all = __builtin_amdgcn_readfirstlane(tid >> 6), wave = all % NW, team = all / NW, lane = tid & 63, g = lane >> 4, li = lane & 15;
    const int h = item % P.heads, slot = item / P.heads;
    const bool packed = P.offsets != nullptr;
    if (packed) clear_rows_of<T>(P, P.out, P.out_f32, P.dc, slot, h, tid, NT);
    Place at;
    if (!at.find(P, slot)) {
        if (SLOPE && tid == 0) P.slope[item] = 0.0;
        return;
    }
    const T *pa = base_of<T>(P.a, packed, at.n_seq, h) + (int64_t)at.lo * P.a.row, *pb = base_of<T>(P.b, packed, at.n_seq, h) + (int64_t)at.lo * P.b.row;
    const T *pc = base_of<T>(P.c, packed, at.n_seq, h) + (int64_t)at.lo * P.c.row;
    const T *pe = SLOPE ? base_of<T>(P.e, packed, at.n_seq, h) + (int64_t)at.lo * P.e.row : nullptr;
    Stage<T, DA, NT, VEC, false> sa, sb;
    Stage<T, DC, NT, VEC, false> sc, se;
    sa.init(la, P.a, tid);
    sb.init(lb, P.b, tid);
    sc.init(lc, P.c, tid);
    if (SLOPE) se.init(le, P.e, tid);
    const auto fetch = [&](int t, int tid) __attribute__((always_inline)) {
        const Next next = at.t1 - t >= CHUNK ? Next{t, CHUNK} : t < at.t1 ? Next{t, at.t1 - t} : Next{at.t0, 1};
        sb.load(pb, P.b, next.t, next.n, tid);
        sa.load(pa, P.a, next.t, next.n, tid);
        sc.load(pc, P.c, next.t, next.n, tid);
        if (SLOPE) se.load(pe, P.e, next.t, next.n, tid);
    };
    if (at.t0 < at.t1) fetch(at.t0, tid);
    __syncthreads();
    Weights<NW * TEAMS> w;
    w.init(P.log_decay[h], P.upd_scale, 0, all, g, li);
    if (all == 0) X::clear_scores(scores, lane);
    const int64_t state_at = ((int64_t)at.n_seq * P.heads + h) * P.da * P.dc;
    X x;
    x.tiles.init(w.lg2, team);
    x.enter(at.segment > 0 ? P.seg + (int64_t)item * P.da * P.dc : P.state_in ? P.state_in + state_at : nullptr, P.st_a, P.st_c, P.da, P.dc, wave, g, li);
    double slope = 0.0;
    const auto chunk = [&](auto rows, int t, int n) __attribute__((always_inline)) {
        typedef decltype(rows) R;
        constexpr bool FULL = R::FULL;
        const int tid = here(tid_), lane = tid & 63, g = lane >> 4, li = lane & 15;
        sb.template store<R>(lb, pb, P.b, t, n, tid);
        sa.template store<R>(la, pa, P.a, t, n, tid);
        sc.template store<R>(lc, pc, P.c, t, n, tid);
        if (SLOPE) se.template store<R>(le, pe, P.e, t, n, tid);
        __syncthreads();
        if (FULL) fetch(t + CHUNK, tid);
#pragma unroll
        for (int m = 0; m < w.MINE; ++m) {
            const int it = w.it[m], jt = w.jt[m];
            if (it >= R::LIVE) continue;
            f32x4 s = X::score(la, lb, it, jt, g, li);
#pragma unroll
            for (int r = 0; r < 4; ++r) s[r] = w.template weigh<R>(s[r], m, r, n, g, li);
            X::keep(s, scores, it, jt, lane);
        }
        if (SLOPE && team == 0) {
            f32x4 *to = (f32x4 *)chunk_states + (((t - at.t0) / CHUNK * NW + wave) * X::TA * X::CT) * 64 + lane;
#pragma unroll
            for (int mt = 0; mt < X::TA; ++mt)
#pragma unroll
                for (int ct = 0; ct < X::CT; ++ct) to[(mt * X::CT + ct) * 64] = x.S[mt][ct];
        }
        phase();
        x.template from_state<R>(la, n, w, g, li);
        if (SLOPE) slope += (double)(x.template dot<R>(le, 1, wave, g, li) * P.out_scale);
        __syncthreads();
        phase();
        x.template columns<R>(lc, wave, g, li);
        x.template from_rows<R, false>(scores, n, P.out_scale, P.out, P.out_f32, (packed ? 0 : (int64_t)at.n_seq * P.rows) + at.lo + t, P.heads, h, P.dc, wave, lane);
        phase();
        x.template advance<R>(lb, n, w, P.upd_scale, 0, g, li);
        __syncthreads();
    };
    int t = at.t0;
    for (; at.t1 - t >= CHUNK; t += CHUNK) chunk(Whole(), t, CHUNK);
    if (at.t1 - t > CHUNK / 2) chunk(Most(), t, at.t1 - t);
    else if (t < at.t1) chunk(Half(), t, at.t1 - t);
    x.leave(at.last && P.state_out && team == 0 ? P.state_out + state_at : nullptr, P.st_a, P.st_c, P.da, P.dc, wave, g, li);
    if (SLOPE) workgroup_sum<NT>(slope, (double *)&lds, P.slope + item, tid);
}

template <typename T, int DA, int DC, int NW, bool VEC, int WAVES> __global__ __launch_bounds__(64 * NW, WAVES) void td_decay_out_kernel(Pass P) {
    __shared__ __align__(16) OutLds<T, DA, DC, NW, false> lds;
    out_sweep<T, DA, DC, NW, 1, VEC, false>(P, P.first + blockIdx.x, lds, nullptr);
}

// out from (a, b, c) and out2 from (e, c, b), rows descending: the gradients of v and k from (k, q, grad_o) and (v, grad_o, q).  SLOPE: the rest of
// the derivative by log g: pairs of rows of one chunk; what a chunk's rows owe to the chunks behind it; and the chunk's own n rows, for every pair with one
// row before and one behind it, which is n g^n <state entering the chunk, its gradient when it leaves>.  TEAMS = 2: NW waves for each of the two
// gradients, at the same time, where one workgroup's LDS or registers fill a compute unit and NW = 4 waves would leave half of each SIMD's places empty.
template <typename T, int DK, int DV, int NW> struct PairLds {
    typedef Stream<T, DK, DV, NW, true> V;
    T k[CHUNK * V::PA], q[CHUNK * V::PA], o[CHUNK * V::PC], v[CHUNK * V::PC];
    typename V::Op scores[2][V::PAIRS * V::TERMS * 64];
};
template <typename T, int DK, int DV, int NW, int TEAMS, bool VEC, bool SLOPE>
__device__ __forceinline__ void pair_sweep(const Pass &P, int item, PairLds<T, DK, DV, NW> &lds, const float *chunk_states) {
    typedef Stream<T, DK, DV, NW, VEC> V;
    typedef Stream<T, DV, DK, NW, VEC> K;
    typedef typename V::Op Op;
    constexpr int NT = 64 * NW * TEAMS;
    T *const lk = lds.k, *const lq = lds.q, *const lo = lds.o, *const lv = lds.v;
    Op *const scores_k = lds.scores[0], *const scores_v = lds.scores[1];
    const int tid_ = here(threadIdx.x), tid = tid_, all = __builtin_amdgcn_readfirstlane(tid >> 6), wave = all % NW, team = all / NW, lane = tid & 63, g = lane >> 4, li = lane & 15;
    const int h = item % P.heads, slot = item / P.heads;
    const bool packed = P.offsets != nullptr;
    if (packed) {
        clear_rows_of<T>(P, P.out, P.out_f32, P.dc, slot, h, tid, NT);
        clear_rows_of<T>(P, P.out2, P.out2_f32, P.da, slot, h, tid, NT);
    }
    Place at;
    if (!at.find(P, slot)) {
        if (SLOPE && tid == 0) P.slope[item] = 0.0;
        return;
    }
    const T *pk = base_of<T>(P.a, packed, at.n_seq, h) + (int64_t)at.lo * P.a.row, *pq = base_of<T>(P.b, packed, at.n_seq, h) + (int64_t)at.lo * P.b.row;
    const T *po = base_of<T>(P.c, packed, at.n_seq, h) + (int64_t)at.lo * P.c.row, *pv = base_of<T>(P.e, packed, at.n_seq, h) + (int64_t)at.lo * P.e.row;
    Stage<T, DK, NT, VEC, true> sk, sq;
    Stage<T, DV, NT, VEC, true> so, sv;
    sk.init(lk, P.a, tid);
    sq.init(lq, P.b, tid);
    so.init(lo, P.c, tid);
    sv.init(lv, P.e, tid);
    const auto fetch = [&](Next next, int tid) __attribute__((always_inline)) {
        sk.load(pk, P.a, next.t, next.n, tid);
        sq.load(pq, P.b, next.t, next.n, tid);
        so.load(po, P.c, next.t, next.n, tid);
        sv.load(pv, P.e, next.t, next.n, tid);
    };
    const int whole = (at.t1 - at.t0) / CHUNK, tail = (at.t1 - at.t0) % CHUNK;
    if (at.t0 < at.t1) fetch(tail ? Next{at.t1 - tail, tail} : Next{at.t1 - CHUNK, CHUNK}, tid);
    __syncthreads();
    Weights<NW> w;
    w.init(P.log_decay[h], P.upd_scale, 1, wave, g, li);
    if (all == 0) {
        V::clear_scores(scores_k, lane);
        V::clear_scores(scores_v, lane);
    }
    const int64_t state_at = ((int64_t)at.n_seq * P.heads + h) * P.da * P.dc;
    const float *from = !at.last ? P.seg + (int64_t)item * P.da * P.dc : P.state_in ? P.state_in + state_at : nullptr;
    double slope = 0.0;
    if constexpr (TEAMS == 2) {
        // One gradient a team: X its stream with rows x, y, z as (a, b, c), SL whether it has the slope's sums too
        const auto one = [&](auto stream, T *lx, T *ly, T *lz, typename V::Op *scores, void *out, int out_f32, int64_t st_x, int64_t st_z, int dx, int dz, auto sums)
                             __attribute__((always_inline)) {
            typedef decltype(stream) X;
            constexpr bool SL = decltype(sums)::value;
            X x;
            x.tiles.init(w.lg2, 0);
            x.enter(from, st_x, st_z, dx, dz, wave, g, li);
            const auto chunk = [&](auto rows, int t, int n, Next next) __attribute__((always_inline)) {
                typedef decltype(rows) R;
                const int tid = here(tid_), lane = tid & 63, g = lane >> 4, li = lane & 15;
                f32x4 F[SL ? X::TA : 1][X::CT];
                if (SL) {
                    const f32x4 *from = (const f32x4 *)chunk_states + (((t - at.t0) / CHUNK * NW + wave) * X::TA * X::CT) * 64 + lane;
#pragma unroll
                    for (int mt = 0; mt < X::TA; ++mt)
#pragma unroll
                        for (int ct = 0; ct < X::CT; ++ct) F[mt][ct] = from[(mt * X::CT + ct) * 64];
                }
                sk.template store<R>(lk, pk, P.a, t, n, tid);
                sq.template store<R>(lq, pq, P.b, t, n, tid);
                so.template store<R>(lo, po, P.c, t, n, tid);
                sv.template store<R>(lv, pv, P.e, t, n, tid);
                __syncthreads();
                fetch(next, tid);
                float sum = 0.0f;
#pragma unroll
                for (int m = 0; m < w.MINE; ++m) {
                    const int it = w.it[m], jt = w.jt[m];
                    if (it >= R::LIVE) continue;
                    f32x4 s = X::score(lx, ly, it, jt, g, li);
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[r] = w.template weigh<R>(s[r], m, r, n, g, li);
                    X::keep(s, scores, it, jt, lane);
                    if (SL) {
                        const f32x4 other = V::score(lk, lq, it, jt, g, li);
#pragma unroll
                        for (int r = 0; r < 4; ++r) sum += w.template pair<R>(m, r, n, g, li) ? (float)w.apart(m, r, g, li) * s[r] * other[r] : 0.0f;
                    }
                }
                const int64_t row0 = (packed ? 0 : (int64_t)at.n_seq * P.rows) + at.lo + t;
                phase();
                x.template from_state<R>(lx, n, w, g, li);
                if (SL) sum += x.template dot<R>(lk, 0, wave, g, li);
                __syncthreads();
                phase();
                x.template columns<R>(lz, wave, g, li);
                x.template from_rows<R, true>(scores, n, 1.0f, out, out_f32, row0, P.heads, h, dz, wave, lane);
                if (SL) {
                    float cross = 0.0f;
#pragma unroll
                    for (int mt = 0; mt < X::TA; ++mt)
#pragma unroll
                        for (int ct = 0; ct < X::CT; ++ct)
#pragma unroll
                            for (int r = 0; r < 4; ++r) cross += F[mt][ct][r] * x.S[mt][ct][r];
                    slope += (double)(sum + (float)n * (R::FULL ? w.whole.hi : power(w.lg2, n)) * cross);
                }
                phase();
                x.template advance<R>(ly, n, w, P.upd_scale, 1, g, li);
                __syncthreads();
            };
            const Next before = whole ? Next{at.t1 - tail - CHUNK, CHUNK} : Next{at.t0, 1};
            if (tail > CHUNK / 2) chunk(Most(), at.t1 - tail, tail, before);
            else if (tail) chunk(Half(), at.t1 - tail, tail, before);
            for (int c = whole - 1; c >= 0; --c) chunk(Whole(), at.t0 + c * CHUNK, CHUNK, c > 0 ? Next{at.t0 + (c - 1) * CHUNK, CHUNK} : Next{at.t0, 1});
            x.leave(at.segment == 0 && P.state_out && team == 1 ? P.state_out + state_at : nullptr, st_x, st_z, dx, dz, wave, g, li);
        };
        // (both ways have the same barriers)
        if (team) one(V(), lk, lq, lo, scores_v, P.out, P.out_f32, P.st_a, P.st_c, P.da, P.dc, Flag<false>());
        else one(K(), lv, lo, lq, scores_k, P.out2, P.out2_f32, P.st_c, P.st_a, P.dc, P.da, Flag<SLOPE>());
    } else {
        V xv;
        K xk;
        xv.tiles.init(w.lg2, 0);
        xk.tiles.init(w.lg2, 0);
        xv.enter(from, P.st_a, P.st_c, P.da, P.dc, wave, g, li);
        xk.enter(from, P.st_c, P.st_a, P.dc, P.da, wave, g, li);
        const auto chunk = [&](auto rows, int t, int n, Next next) __attribute__((always_inline)) {
            typedef decltype(rows) R;
            constexpr bool FULL = R::FULL;
            const int tid = here(tid_), lane = tid & 63, g = lane >> 4, li = lane & 15;
            f32x4 F[SLOPE ? K::TA : 1][K::CT];         // the state that entered this chunk ascending
            if (SLOPE) {
                const f32x4 *from = (const f32x4 *)chunk_states + (((t - at.t0) / CHUNK * NW + wave) * K::TA * K::CT) * 64 + lane;
#pragma unroll
                for (int mt = 0; mt < K::TA; ++mt)
#pragma unroll
                    for (int ct = 0; ct < K::CT; ++ct) F[mt][ct] = from[(mt * K::CT + ct) * 64];
            }
            sk.template store<R>(lk, pk, P.a, t, n, tid);
            sq.template store<R>(lq, pq, P.b, t, n, tid);
            so.template store<R>(lo, po, P.c, t, n, tid);
            sv.template store<R>(lv, pv, P.e, t, n, tid);
            __syncthreads();
            fetch(next, tid);
            float sum = 0.0f;
#pragma unroll
            for (int m = 0; m < w.MINE; ++m) {
                const int it = w.it[m], jt = w.jt[m];
                if (it >= R::LIVE) continue;
                f32x4 sv = V::score(lk, lq, it, jt, g, li), sk = K::score(lv, lo, it, jt, g, li);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    sv[r] = w.template weigh<R>(sv[r], m, r, n, g, li);
                    if (SLOPE) sum += w.template pair<R>(m, r, n, g, li) ? (float)w.apart(m, r, g, li) * sv[r] * sk[r] : 0.0f;
                    sk[r] = w.template weigh<R>(sk[r], m, r, n, g, li);
                }
                V::keep(sv, scores_v, it, jt, lane);
                K::keep(sk, scores_k, it, jt, lane);
            }
            const int64_t row0 = (packed ? 0 : (int64_t)at.n_seq * P.rows) + at.lo + t;
            phase();
            xk.template from_state<R>(lv, n, w, g, li);
            if (SLOPE) sum += xk.template dot<R>(lk, 0, wave, g, li);
            __syncthreads();
            phase();
            xk.template columns<R>(lq, wave, g, li);
            xk.template from_rows<R, true>(scores_k, n, 1.0f, P.out2, P.out2_f32, row0, P.heads, h, P.da, wave, lane);
            if (SLOPE) {
                float cross = 0.0f;
#pragma unroll
                for (int mt = 0; mt < K::TA; ++mt)
#pragma unroll
                    for (int ct = 0; ct < K::CT; ++ct)
#pragma unroll
                        for (int r = 0; r < 4; ++r) cross += F[mt][ct][r] * xk.S[mt][ct][r];
                slope += (double)(sum + (float)n * (R::FULL ? w.whole.hi : power(w.lg2, n)) * cross);
            }
            phase();
            xk.template advance<R>(lo, n, w, P.upd_scale, 1, g, li);
            phase();
            xv.template from_state<R>(lk, n, w, g, li);
            phase();
            xv.template columns<R>(lo, wave, g, li);
            xv.template from_rows<R, true>(scores_v, n, 1.0f, P.out, P.out_f32, row0, P.heads, h, P.dc, wave, lane);
            phase();
            xv.template advance<R>(lq, n, w, P.upd_scale, 1, g, li);
            __syncthreads();
        };
        const Next before = whole ? Next{at.t1 - tail - CHUNK, CHUNK} : Next{at.t0, 1};
        if (tail > CHUNK / 2) chunk(Most(), at.t1 - tail, tail, before);
        else if (tail) chunk(Half(), at.t1 - tail, tail, before);
        for (int c = whole - 1; c >= 0; --c) chunk(Whole(), at.t0 + c * CHUNK, CHUNK, c > 0 ? Next{at.t0 + (c - 1) * CHUNK, CHUNK} : Next{at.t0, 1});
        xv.leave(at.segment == 0 && P.state_out ? P.state_out + state_at : nullptr, P.st_a, P.st_c, P.da, P.dc, wave, g, li);
    }
    if (SLOPE) workgroup_sum<NT>(slope, (double *)&lds, P.slope + item, tid);
}

// The gradients of one (slot, head) after another: that of q with Q's rows ascending, those of k and v with R's descending, right behind each other
// so that the second reading of q, k, v and grad_o (and, for the slope, of the states entering the chunks, in a place of the
// workgroup's own: `held` floats) comes from the caches.
template <typename T, int DK, int DV, int NW, int TEAMS, bool VEC, bool SLOPE, int WAVES>
__global__ __launch_bounds__(64 * NW * TEAMS, WAVES) void td_decay_backward_kernel(Pass Q, Pass R, float *chunk_states, int64_t held, int ascending, int descending) {
    __shared__ __align__(16) union {
        OutLds<T, DV, DK, NW, SLOPE> out;
        PairLds<T, DK, DV, NW> pair;
    } lds;
    float *mine = chunk_states + blockIdx.x * held;
    for (unsigned item = blockIdx.x; item < (unsigned)(Q.slots * Q.heads); item += gridDim.x) {
        if (ascending) out_sweep<T, DV, DK, NW, TEAMS, VEC, SLOPE>(argument<Pass>(0), item, lds.out, mine);
        __syncthreads();
        if (descending) pair_sweep<T, DK, DV, NW, TEAMS, VEC, SLOPE>(argument<Pass>(sizeof(Pass)), item, lds.pair, mine);
        __syncthreads();
    }
}

}  // namespace decay
