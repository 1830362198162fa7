// Products of 8-bit integers with a scale for each row of the first operand and each column of the second, on the assembly tile:
//   out[m, n] = a_scale[m] * b_scale[n] * sum over k of a[m, k] * b[n, k],  rows of one group's matrix or jagged over many.
// v_mfma_i32_16x16x64_i8 takes 16 bytes of each operand from a lane, as the bf16 product does, so the tile's copies, LDS layout and loop are
// those of the 16-bit tile with twice as many values in a byte of everything (gen_tile_asm.py); sums are exact, the scales are applied in fp32
// in the epilogue, one rounding follows.  Tile list, launch order and cut tiles are the 16-bit product's.
//   8192 x 14336 x 4096 bf16 out                 354 us, 2.7 POP/s.  A K tile of 128 takes 1.37 us (3.1 POP/s); what is left is a tile's prologue and its
//                                                stores, which all compute units make at once: 10 us a round
//   8 of 128 experts, 4001 tokens, 2048 -> 2 x 768   164 us with SwiGLU in the epilogue, 768 -> 2048 142 to 148 to fp32 (bf16 124): 22 and 8 us of K tiles and the
//                                                same 10 of prologue and stores.  128-row tiles throughout, or groups in another order: no faster
#define GMM_TILE_INT8
#include "gmm_asm.h"

namespace {

template <int OUT_F32, int F16>
int launch(const GmmInt8Params& p, hipStream_t stream) {
  hipLaunchKernelGGL((gmm_asm_kernel<0, 0, OUT_F32, F16, 0, ORDER_PLAIN, GmmInt8Params>), dim3(p.num_wg), dim3(256), 0, stream, p);
  return hipGetLastError() == hipSuccess ? 0 : 1;
}

void set_tiles(GmmInt8Params& p, int num_cus) {
  // as for 16-bit products: 256-row tiles unless they would not fill four rounds, and then group by group
  const int64_t tn = gmm_cdiv(p.N, 256);
  const int64_t est = p.jag == GMM_JAG_M ? (int64_t(p.M) / 256 + gmm_min(p.G, p.M)) * tn : int64_t(p.G) * gmm_cdiv(p.M, 256) * tn;
  p.tall = est < 4 * int64_t(num_cus) ? 128 : 256;
  p.shrt = 64;
  p.group_major = p.tall == 128;
  p.xcd_remap = 1;
  p.align = 1;
  plan(p, GmmLayout{true, true}, GMM_CFG_ASM_256x256, num_cus);
}

}  // namespace

bool gmm_int8_tile_uses_workspace(GmmInt8Params p, int num_cus) {
  set_tiles(p, num_cus);
  return p.ws_parts > 0;
}

int gmm_launch_int8_tile(GmmInt8Params p, int out_dtype, int num_cus, hipStream_t stream) {
  set_tiles(p, num_cus);
  if (p.act) {
    hipLaunchKernelGGL((gmm_asm_kernel<0, 0, 1, 2, 4, ORDER_PLAIN, GmmInt8Params>), dim3(p.num_wg), dim3(256), 0, stream, p);
    return hipGetLastError() == hipSuccess ? 0 : 1;
  }
  if (out_dtype == GMM_DT_BF16) return launch<0, 2>(p, stream);
  if (out_dtype == GMM_DT_F16) return launch<0, 3>(p, stream);
  return launch<1, 2>(p, stream);
}
