// "attn" module: the part of attention behind a shared prefix for sequences of few rows (attn_shared.hip has the description).
// Bound: latency, as where few keys are seen by attention itself: 128 sequences of a token with up to 600 keys of their own 23 us, 4 waves of each work-group two
// or three steps of 32 keys each.
#include "attn_few.inc"

// -DFINE=1: blocks of one or two tokens, a scale for each key; 0: a scale for each four
#define FEW(HD, RT, PACK, FINE, W, F)                                                                                                                         \
  extern "C" __global__ __launch_bounds__(256, W) void attn_part_few__HD##HD##_RT##RT##_PACK##PACK##_FINE##FINE##_FORM##F(                                    \
      const float* q, int ldq, int q_off, const int8_t* kq, const int8_t* vq, const float* ks, const float* vs, int pages, int ps, int bs, const int* rows,   \
      const int* lens, const int* table, int ldt, int T, int max_rows, int heads, int kvh, float scale, float cap2, int window, const float* slopes,          \
      const int* prefix, const int* first, const int* groups, const int* shared, int n, int places, int per, char* room, size_t at, int nsplit, int least,    \
      int vec) {                                                                                                                                              \
    const int g = attn::group_of(groups, n, blockIdx.x / kvh);                                                                                                \
    few_body<HD, RT, PACK, FINE, (F & 1) != 0, (F & 2) != 0, true>(q, ldq, q_off, kq, vq, ks, vs, pages, ps, bs, rows, lens, table, ldt, T, max_rows, heads,  \
                                                                   kvh, nullptr, 0, 0, scale, cap2, window, slopes, prefix, first, (float*)(room + at),       \
                                                                   nullptr, nsplit, least, vec, g < 0 ? 0 : max(shared[g], 0), places, per);                  \
  }
#define FEW4(HD, RT, PACK, FINE, W) FEW(HD, RT, PACK, FINE, W, 0) FEW(HD, RT, PACK, FINE, W, 1) FEW(HD, RT, PACK, FINE, W, 2) FEW(HD, RT, PACK, FINE, W, 3)
// W, WF: waves a SIMD that the registers are held to (WF: with a scale for each key)
#define FEWF(HD, RT, PACK, W, WF) FEW4(HD, RT, PACK, 0, W) FEW4(HD, RT, PACK, 1, WF)
FEWF(64, 1, 1, 4, 4)
FEWF(64, 1, 0, 4, 3)
FEWF(64, 2, 0, 3, 2)
FEWF(128, 1, 1, 3, 3)
FEWF(128, 1, 0, 3, 2)
FEWF(128, 2, 0, 2, 1)
FEWF(256, 1, 1, 2, 2)   // (two row tiles of 256 values do not fit a wave's registers: such rows go to attn_many)
FEWF(256, 1, 0, 2, 1)
