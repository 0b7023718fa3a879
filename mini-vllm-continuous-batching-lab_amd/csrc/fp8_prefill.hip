// Prefill attention over the 8-bit KV cache (format: mv_fp8.h): the 16-bit
// kernels (mv_prefill16.h) with the prefix's codes turned into 16-bit values on
// their way into LDS. What a code stands for is a number of the model's type, so
// the result is the 16-bit kernel's over the dequantised pool, bit for bit. Bound
// as there, by issue slots beside the MFMAs; the conversion takes 5-11 % (measured
// beside Fp8SubTile): 8 x (300-2900 + 100-900) at 28 / 4 x 128 124 us, 844 TFLOP/s.
#include "mv_prefill16.h"

namespace mv {
namespace {

template <int DTYPE, int D, bool WIDE, typename BT>
__global__ __launch_bounds__(512) void fp8_prefill_kernel(PrefillArgs a) {
  prefill16<Prefill16Traits<DTYPE, D, WIDE ? 8 : 4, WIDE ? 1 : 2, true>, BT>(a);
}

template <int DTYPE, int D>
void launch(const PrefillArgs& a, int groups, bool bt_i64, bool wide, hipStream_t s) {
  if (wide) {
    if (bt_i64) fp8_prefill_kernel<DTYPE, D, true, int64_t><<<groups, 512, 0, s>>>(a);
    else fp8_prefill_kernel<DTYPE, D, true, int32_t><<<groups, 512, 0, s>>>(a);
  } else {
    if (bt_i64) fp8_prefill_kernel<DTYPE, D, false, int64_t><<<groups, 512, 0, s>>>(a);
    else fp8_prefill_kernel<DTYPE, D, false, int32_t><<<groups, 512, 0, s>>>(a);
  }
}

}  // namespace

int launch_prefill_fp8(const PrefillArgs& a, int head_dim, int dtype, int groups, bool bt_i64, bool wide,
                       hipStream_t s) {
  if (dtype == MV_DTYPE_F16) {
    if (head_dim == 64) launch<MV_DTYPE_F16, 64>(a, groups, bt_i64, wide, s);
    else launch<MV_DTYPE_F16, 128>(a, groups, bt_i64, wide, s);
  } else {
    if (head_dim == 64) launch<MV_DTYPE_BF16, 64>(a, groups, bt_i64, wide, s);
    else launch<MV_DTYPE_BF16, 128>(a, groups, bt_i64, wide, s);
  }
  return check_launch("mv_fp8_paged_prefill");
}

}  // namespace mv
