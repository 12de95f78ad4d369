// "attn" module: attention of many rows over the 8-bit cache -- prompts and chunks behind a context.
//
// Per kv head the rows are the sequence's tokens times the query heads that share it (row = token * group + head), 128 to a
// work-group, 32 to a wave.  KT keys at a time are brought into LDS as f16 -- the eight-bit values exactly, converted once for
// the four waves --, the keys as they lie, the values with tokens and columns exchanged; the next tile's bytes are on their
// way meanwhile.
//
//   S^T = K Q^T   32 x 32 x 16 products, A = 32 keys from LDS, B = 32 rows held in registers: a lane has 16 keys' scores of one row
//   O^T += V^T P^T  B = the weights just as the scores' product left them (a lane's keys of a slot of 16 are 4 h + 0..3 and
//                  8 + 4 h + 0..3, so the values' tokens lie in that order in LDS): no weight goes through LDS
//
// A row's maximum and sum are its lane's own, but for the two halves of the wave, which meet only where the reference is set
// anew.  Rows and weights are split into two f16 (22 bits of the f32 value, a row on its own power of two; the sums are those of f32
// rows to about 2^-22), so the matrix pipe does twice the products of plain f16 rows: most of the time of long prompts.
//
// Measured, 32 query heads over 8 of 128 values: 8192 rows behind 808 keys, causal, 1109 - 1172 us by the card = 562 - 593 TFLOP/s of
// attention, 1124 - 1186 of products (a large f16 matrix product of the library: 1211).  The matrix pipe is busy 62 % of 2.05 million
// cycles, which makes about 1.85 GHz: like the library's product the launch runs below the card's highest clock, and the third of
// the cycles in which no product is under way (a tile's meeting, weights that are not done when they are wanted) costs less time
// than it would at that.  On the way there: 2000 us with the tiles' rows 8 and 16 bytes apart in the same banks (conflicts in 64 %
// of the LDS's cycles, now 0.3 %); 1303 with the rows that see the most keys first; 1141 with no wait for a page's number inside the
// loop; the last 7 to 10 with keys and values as global loads (through pointers of no known address space they counted among
// the LDS reads, and every operand was waited for with them).
// Rows of several documents (1333 rows, 40 heads): 67 us, the matrix pipe busy 22 %: most tiles are one document's end.
// Spills, all before and behind the loop: 4 and 8 registers of heads of 256 with a scale for each few keys and a cap, 9 of eight waves with
// a distance.
#include "attn_many.inc"

// -DFINE=1: blocks of less than 32 tokens; -DW8: work-groups of eight waves, 256 rows, one a compute unit: a tile is staged once for
// twice the rows (for blocks of 32 tokens and more: with a scale for each key its loop does not fit the registers)
#define MANY(NAME, HD, KT, NW, W, FINE, F)                                                                                                                      \
  extern "C" __global__ __launch_bounds__(64 * NW, W) void NAME(                                                                                                \
      const float* q, int ldq, int q_off, const int8_t* kq, const int8_t* vq, const float* ks, const float* vs, int pages, int ps, int bs, const int* rows,     \
      const int* lens, const int* table, int ldt, int T, int max_rows, int heads, int kvh, float* out, int ldo, int o_off, float scale, float cap2, int window, \
      const float* slopes, const int* prefix, const int* first, float* ws, int nsplit, int tiles, int vec) {                                                    \
    many_body<HD, KT, NW, FINE, (F & 1) != 0, (F & 2) != 0>(q, ldq, q_off, kq, vq, ks, vs, pages, ps, bs, rows, lens, table, ldt, T, max_rows, heads, kvh, out, \
                                                            ldo, o_off, scale, cap2, window, slopes, prefix, first, ws, nsplit, tiles, vec);                    \
  }
#define MANY4(HD, KT, NW, W, FINE, S)                              \
  MANY(attn_many__HD##HD##_FINE##FINE##_FORM0##S, HD, KT, NW, W, FINE, 0) \
  MANY(attn_many__HD##HD##_FINE##FINE##_FORM1##S, HD, KT, NW, W, FINE, 1) \
  MANY(attn_many__HD##HD##_FINE##FINE##_FORM2##S, HD, KT, NW, W, FINE, 2) \
  MANY(attn_many__HD##HD##_FINE##FINE##_FORM3##S, HD, KT, NW, W, FINE, 3)
MANY4(64, 64, 4, 2, 0, )
MANY4(64, 64, 4, 2, 1, )
MANY4(128, 32, 4, 2, 0, )
MANY4(128, 32, 4, 2, 1, )
MANY4(128, 64, 8, 2, 0, _W81)
MANY4(256, 32, 4, 1, 0, )
MANY4(256, 32, 4, 1, 1, )
