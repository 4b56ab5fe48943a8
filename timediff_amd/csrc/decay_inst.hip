// One object per (element type, kernel) of decay attention: TD_INST_BF16 0 or 1, TD_INST_KIND as decay::Kind.
#include "decay_chunk.h"

using namespace decay;

#define TD_CAT_(a, b, c) a##b##_##c
#define TD_CAT(a, b, c) TD_CAT_(a, b, c)

namespace {

#if TD_INST_BF16
typedef __bf16 T;
#else
typedef float T;
#endif

// A wave for each 16 columns of the output (backward: of the narrower of its two outputs); the bfloat16 forward pass of 128 x 128 takes 32 columns
// a wave, so that two workgroups share a compute unit.  Backward passes of four waves of which a compute unit holds one workgroup take a second team of
// four.  Waves a SIMD that a kernel is built for: four in the bfloat16 forward pass of 64 x 128, three in forward passes up to 64 x 64 (float32
// reaches two), else two (float32 forward of 128 x 64, with one workgroup of four waves in LDS: one).  At two the backward passes of aligned tensors
// with log_decay's gradient spill, of 128 x 128 199 registers (bfloat16) and 475 (float32), of float32 128 x 64 253, and so does that of float32
// 128 x 128 with fixed decays, 179; the others spill 50 or fewer.  (Odd addresses: 134, 143, 131, 18.)  Measured with 16 sequences of 1024
// rows, 8 heads, unless said otherwise:
//   forward, bfloat16: 128 x 128 4 waves of 32 columns 95 us, 8 of 16 102; 64 x 128 8 waves, 4 a SIMD 59, 4 waves 61;
//   forward, float32 (LDS holds one workgroup): 128 x 128, 64 sequences, 8 waves 418 us, 4 waves 824;
//   backward, bfloat16 (learned / fixed decays): 128 x 128 8 waves 370 / 226, 4 waves 368 / 259; 64 x 128 two teams 170 / 159, one 193 / 180;
//   64 x 64, 2048 sequences of 272 rows: two workgroups of one team 1.07 / 0.94 ms, of two teams 1.43 / 1.27, three of one 1.60 / 0.92;
//   backward, float32: 64 x 64 two teams 197 / 180, one 202 / 190; 64 x 128 335 / 310 and 419 / 386.
template <bool VEC, int DA, int DC> int launch(const Work &w, hipStream_t st) {
    constexpr int size = DA + DC, NW = TD_INST_KIND == 0 && TD_INST_BF16 && size == 256 ? 4 : (TD_INST_KIND < 3 ? DC : DA < DC ? DA : DC) / 16;
    const Pass &P = w.p;
#if TD_INST_KIND < 3
    launch_parts(P, (int64_t)P.slots * P.heads, 64 * NW, [&](const Pass &P, dim3 grid) {
#if TD_INST_KIND == 0
        hipLaunchKernelGGL((td_decay_out_kernel<T, DA, DC, NW, VEC, size <= 128 ? 3 : TD_INST_BF16 && size < 256 && DC == 128 ? 4 : 2>), grid, dim3(64 * NW), 0, st, P);
#else
        hipLaunchKernelGGL((td_decay_sum_kernel<T, DA, DC, NW, VEC, TD_INST_KIND == 2, 4>), grid, dim3(64 * NW), 0, st, P);
#endif
    });
#else
    const int64_t held = (int64_t)((P.seg_len + CHUNK - 1) / CHUNK) * DA * DC;
    constexpr int TEAMS = NW == 4 && (!TD_INST_BF16 || size > 128) ? 2 : 1;
    hipLaunchKernelGGL((td_decay_backward_kernel<T, DA, DC, NW, TEAMS, VEC, TD_INST_KIND == 4, 2>), dim3((unsigned)w.groups), dim3(64 * NW * TEAMS), 0, st, w.p, w.r,
                       w.chunk_states, held, w.ascending, w.descending);
#endif
    TD_LAUNCH_CHECK();
    return TD_OK;
}

}  // namespace

// Sizes, strides or addresses that are not multiples of 16 bytes have kernels of their own, of the same sizes (in the square that holds them
// 41 x 101 and 101 x 41 take longer; 16 sequences of 1024 rows, 8 heads, in rectangles and in squares: backward, bfloat16 432 and 458 us, 616 and 639;
// float32 458 and 589, 769 and 790; forward, bfloat16 114 and 156, 188 and 183; float32 134 and 146, 189 and 180).
int TD_CAT(td_decay_launch_, TD_INST_BF16, TD_INST_KIND)(const Work &w, int vec, hipStream_t st) {
    const Pass &P = TD_INST_KIND < 3 ? w.p : w.r;          // backward: (da, dc) = (dk, dv)
    const int most = P.da > P.dc ? P.da : P.dc;
    if (most <= 32) return vec ? launch<true, 32, 32>(w, st) : launch<false, 32, 32>(w, st);
    if (most <= 64) return vec ? launch<true, 64, 64>(w, st) : launch<false, 64, 64>(w, st);
    if (P.da <= 64) return vec ? launch<true, 64, 128>(w, st) : launch<false, 64, 128>(w, st);
    if (P.dc <= 64) return vec ? launch<true, 128, 64>(w, st) : launch<false, 128, 64>(w, st);
    return vec ? launch<true, 128, 128>(w, st) : launch<false, 128, 128>(w, st);
}
