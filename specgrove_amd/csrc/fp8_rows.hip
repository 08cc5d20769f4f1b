// Rows in e4m3 with a scale for each row and 128 columns, made by what produces
// the rows: the rows as they are, residual add + RMSNorm, SiLU(gate) * up.
//
// A block x of 128 columns with m = max(max |x|, 2^-100) has the scale m / 448
// and the codes e4m3(x * (448 / m)): one division each for the block, and the
// largest code is 448, the largest finite value.  The floor keeps 448 / m finite;
// a block below it rounds towards 0.  fp32 throughout; the one rounding to fewer
// bits is the code's (the sum of the residual add, which stays in memory as bf16,
// is rounded before its norm).  The maximum is taken over the bits of |x|, which
// order as integers with infinities and NaNs above, so that those reach the scale.
//
// Bound by HBM: 16-byte loads, 8 values a lane; 16 lanes hold a block, so its
// maximum takes four lane moves; 8-byte stores of codes.  Columns from K up to the
// next multiple of 128 are written as zeros.  2048 rows: SiLU * up of 12288 columns
// 27 us, 4.6 TB/s (39 with a division in the SiLU and exchanges through the LDS);
// add + RMSNorm of 4096 with its sum 13 us, 4.5 TB/s.
#include <algorithm>

#include "sg_common.h"

namespace sg {
namespace {

constexpr int kThreads = 256;
constexpr int kBlock = 128;                // columns of a scale
constexpr int kPart = 8 * kThreads;        // columns of a workgroup's step
constexpr uint32_t kTinyBits = 0x0d800000u;  // 2^-100

struct Pair {
  float lo, hi;
};
__device__ __forceinline__ Pair unpack(uint32_t v) {
  return {__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)};
}

// a / (1 + exp(-a)), with the exponential of -|a| so that the divisor lies in [1, 2]:
// the reciprocal instruction (1 ulp there) serves, where the division's ten
// instructions took half of the kernel's issue time.
__device__ __forceinline__ float silu(float a) {
  const float e = expf(-fabsf(a));
  return (a < 0.0f ? a * e : a) * __builtin_amdgcn_rcpf(1.0f + e);
}

struct RowsOut {
  unsigned char* codes;
  int64_t code_stride;
  float* scales;
  int64_t scale_stride;
};

// Columns e .. e+7 of row `row` (e a multiple of 8 below Kp); the 16 lanes of the
// block call together.
__device__ __forceinline__ void store_block(const RowsOut& out, int64_t row, int e,
                                            const float (&x)[8]) {
  uint32_t bits = 0u;
#pragma unroll
  for (int k = 0; k < 8; ++k) bits = max(bits, __float_as_uint(x[k]) & 0x7fffffffu);
  bits = max(bits, lane_swap<kSwap1>(bits));
  bits = max(bits, lane_swap<kSwap2>(bits));
  bits = max(bits, lane_swap<kMirror8>(bits));
  bits = max(bits, lane_swap<kMirror16>(bits));
  const float m = __uint_as_float(max(bits, kTinyBits));
  const float r = 448.0f / m;
  uint32_t w[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * k] * r, x[4 * k + 1] * r, 0, false);
    v = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * k + 2] * r, x[4 * k + 3] * r, v, true);
    w[k] = static_cast<uint32_t>(v);
  }
  *reinterpret_cast<uint2*>(out.codes + row * out.code_stride + e) = make_uint2(w[0], w[1]);
  if (e % kBlock == 0) out.scales[(e / kBlock) * out.scale_stride + row] = m / 448.0f;
}

// kSilu: x is [R, 2 columns], gate then up.  A workgroup takes kPart columns of
// one row (parts = workgroups a row).
template <bool kSilu>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const uint16_t* __restrict__ x,
                                                            int64_t x_stride, int columns,
                                                            int padded, RowsOut out,
                                                            uint32_t parts, int64_t items) {
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t row = item / parts;
    const int part = static_cast<int>(item - row * parts);
    const int e = part * kPart + 8 * static_cast<int>(threadIdx.x);
    if (e >= padded) continue;
    const bool live = e < columns;
    const uint16_t* src = x + row * x_stride + e;
    const uint4 g = live ? *reinterpret_cast<const uint4*>(src) : make_uint4(0u, 0u, 0u, 0u);
    const uint32_t gv[4] = {g.x, g.y, g.z, g.w};
    float v[8];
    if constexpr (kSilu) {
      const uint4 u =
          live ? *reinterpret_cast<const uint4*>(src + columns) : make_uint4(0u, 0u, 0u, 0u);
      const uint32_t uv[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const Pair a = unpack(gv[k]), b = unpack(uv[k]);
        v[2 * k] = silu(a.lo) * b.lo;
        v[2 * k + 1] = silu(a.hi) * b.hi;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const Pair a = unpack(gv[k]);
        v[2 * k] = a.lo;
        v[2 * k + 1] = a.hi;
      }
    }
    store_block(out, row, e, v);
  }
}

// One row per workgroup, kChunks chunks of 8 columns a thread (as
// add_rmsnorm_kernel: every load of the row is issued before the first is used).
template <int kChunks, bool kResidual>
__global__ __launch_bounds__(kThreads) void add_rmsnorm_fp8_kernel(
    const uint16_t* __restrict__ x, const uint16_t* __restrict__ residual,
    const uint16_t* __restrict__ weight, uint16_t* __restrict__ residual_out, int hidden,
    int padded, int64_t x_stride, int64_t res_stride, int64_t res_out_stride, float eps,
    RowsOut out) {
  __shared__ float scratch[kThreads / 64];
  const int64_t row = blockIdx.x;
  const uint16_t* xr = x + row * x_stride;
  const uint16_t* rr = residual + row * res_stride;
  uint4 s[kChunks], b[kChunks], w[kChunks];
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    const int e = 8 * (threadIdx.x + c * kThreads);
    const bool live = e < hidden;
    s[c] = live ? *reinterpret_cast<const uint4*>(xr + e) : make_uint4(0u, 0u, 0u, 0u);
    if (kResidual)
      b[c] = live ? *reinterpret_cast<const uint4*>(rr + e) : make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    const int e = 8 * (threadIdx.x + c * kThreads);
    w[c] = e < hidden ? *reinterpret_cast<const uint4*>(weight + e) : make_uint4(0u, 0u, 0u, 0u);
  }
  float ss = 0.0f;
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    uint32_t v[4] = {s[c].x, s[c].y, s[c].z, s[c].w};
    if (kResidual) {
      const uint32_t bv[4] = {b[c].x, b[c].y, b[c].z, b[c].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const Pair p = unpack(v[k]), q = unpack(bv[k]);
        v[k] = pack_bf16x2(p.lo + q.lo, p.hi + q.hi);
      }
      s[c] = make_uint4(v[0], v[1], v[2], v[3]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const Pair p = unpack(v[k]);
      ss += p.lo * p.lo + p.hi * p.hi;
    }
  }
  if (residual_out != nullptr) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int e = 8 * (threadIdx.x + c * kThreads);
      if (e < hidden)
        *reinterpret_cast<uint4*>(residual_out + row * res_out_stride + e) = s[c];
    }
  }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) ss += __shfl_xor(ss, d);
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = ss;
  __syncthreads();
  float total = 0.0f;
#pragma unroll
  for (int k = 0; k < kThreads / 64; ++k) total += scratch[k];
  const float r = 1.0f / sqrtf(total / static_cast<float>(hidden) + eps);
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    const int e = 8 * (threadIdx.x + c * kThreads);
    if (e >= padded) continue;
    const uint32_t v[4] = {s[c].x, s[c].y, s[c].z, s[c].w};
    const uint32_t wv[4] = {w[c].x, w[c].y, w[c].z, w[c].w};
    float n[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const Pair p = unpack(v[k]), q = unpack(wv[k]);
      n[2 * k] = p.lo * r * q.lo;
      n[2 * k + 1] = p.hi * r * q.hi;
    }
    store_block(out, row, e, n);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check_out(const SgFp8RowsOut* out, int num_rows, int padded) {
  SG_REQUIRE(out != nullptr, "null SgFp8RowsOut");
  SG_REQUIRE(out->codes_dev && out->scales_dev, "null device pointer");
  SG_REQUIRE(out->code_stride >= padded && out->code_stride % 16 == 0 &&
                 aligned16(out->codes_dev),
             "codes must be 16-byte aligned, their stride a multiple of 16 that covers a row "
             "padded to 128 columns");
  SG_REQUIRE(out->scale_stride >= num_rows, "scale_stride must cover the rows");
  return SG_OK;
}

RowsOut rows_out(const SgFp8RowsOut& o) {
  return {static_cast<unsigned char*>(o.codes_dev), o.code_stride, o.scales_dev, o.scale_stride};
}

int padded_columns(int columns) { return (columns + kBlock - 1) / kBlock * kBlock; }

template <bool kSilu>
int launch_quantize(const void* x, int64_t x_stride, int num_rows, int columns,
                    const SgFp8RowsOut* out, sg_stream_t stream) {
  const int padded = padded_columns(columns);
  if (const int rc = check_out(out, num_rows, padded)) return rc;
  const uint32_t parts = (static_cast<uint32_t>(padded) + kPart - 1) / kPart;
  const int64_t items = static_cast<int64_t>(num_rows) * parts;
  quantize_kernel<kSilu>
      <<<dim3(static_cast<unsigned>(std::min<int64_t>(items, 1 << 20))), dim3(kThreads), 0,
         static_cast<hipStream_t>(stream)>>>(static_cast<const uint16_t*>(x), x_stride, columns,
                                             padded, rows_out(*out), parts, items);
  SG_LAUNCH_CHECK();
  return SG_OK;
}

}  // namespace
}  // namespace sg

extern "C" int sg_fp8_quantize_rows(const void* x_dev, int64_t x_stride, int32_t num_rows,
                                    int32_t columns, const SgFp8RowsOut* out,
                                    sg_stream_t stream) {
  using namespace sg;
  clear_error();
  SG_REQUIRE(num_rows >= 0 && columns >= 8 && columns % 8 == 0 && columns <= (1 << 24),
             "columns must be a multiple of 8 in [8, 2^24]");
  if (num_rows == 0) return SG_OK;
  SG_REQUIRE(x_dev != nullptr, "null device pointer");
  SG_REQUIRE(x_stride >= columns && x_stride % 8 == 0 && aligned16(x_dev),
             "x must be 16-byte aligned, its row stride a multiple of 8 that covers a row");
  return launch_quantize<false>(x_dev, x_stride, num_rows, columns, out, stream);
}

extern "C" int sg_silu_mul_fp8(const void* gate_up_dev, int64_t gate_up_row_stride,
                               int32_t num_rows, int32_t intermediate, const SgFp8RowsOut* out,
                               sg_stream_t stream) {
  using namespace sg;
  clear_error();
  SG_REQUIRE(num_rows >= 0 && intermediate >= 8 && intermediate % 8 == 0 &&
                 intermediate <= (1 << 24),
             "intermediate must be a multiple of 8 in [8, 2^24]");
  if (num_rows == 0) return SG_OK;
  SG_REQUIRE(gate_up_dev != nullptr, "null device pointer");
  SG_REQUIRE(gate_up_row_stride >= 2 * static_cast<int64_t>(intermediate) &&
                 gate_up_row_stride % 8 == 0 && aligned16(gate_up_dev),
             "gate_up must be 16-byte aligned, its row stride a multiple of 8 that covers a row");
  return launch_quantize<true>(gate_up_dev, gate_up_row_stride, num_rows, intermediate, out,
                               stream);
}

extern "C" int sg_add_rmsnorm_fp8(const SgAddRmsNormArgs* args, const SgFp8RowsOut* out,
                                  sg_stream_t stream) {
  using namespace sg;
  clear_error();
  SG_REQUIRE(args != nullptr, "null args");
  const SgAddRmsNormArgs& a = *args;
  SG_REQUIRE(a.num_rows >= 0, "num_rows must be non-negative");
  SG_REQUIRE(a.hidden >= 8 && a.hidden % 8 == 0 && a.hidden <= 8 * 4 * kThreads,
             "hidden must be a multiple of 8 in [8, 8192]");
  if (a.num_rows == 0) return SG_OK;
  SG_REQUIRE(a.x_dev && a.weight_dev, "null device pointer");
  SG_REQUIRE((a.x_stride | (a.residual_dev ? a.residual_stride : 0) |
              (a.residual_out_dev ? a.residual_out_stride : 0)) % 8 == 0,
             "row strides must be multiples of 8 elements");
  SG_REQUIRE(aligned16(a.x_dev) && aligned16(a.weight_dev) &&
                 (!a.residual_dev || aligned16(a.residual_dev)) &&
                 (!a.residual_out_dev || aligned16(a.residual_out_dev)),
             "tensors must be 16-byte aligned");
  const int padded = padded_columns(a.hidden);
  if (const int rc = check_out(out, a.num_rows, padded)) return rc;
  auto go = [&](auto kernel) {
    kernel<<<dim3(a.num_rows), dim3(kThreads), 0, static_cast<hipStream_t>(stream)>>>(
        static_cast<const uint16_t*>(a.x_dev), static_cast<const uint16_t*>(a.residual_dev),
        static_cast<const uint16_t*>(a.weight_dev), static_cast<uint16_t*>(a.residual_out_dev),
        a.hidden, padded, a.x_stride, a.residual_stride, a.residual_out_stride, a.eps,
        rows_out(*out));
  };
  const bool res = a.residual_dev != nullptr;
  switch ((padded + 8 * kThreads - 1) / (8 * kThreads)) {
    case 1: res ? go(add_rmsnorm_fp8_kernel<1, true>) : go(add_rmsnorm_fp8_kernel<1, false>); break;
    case 2: res ? go(add_rmsnorm_fp8_kernel<2, true>) : go(add_rmsnorm_fp8_kernel<2, false>); break;
    case 3: res ? go(add_rmsnorm_fp8_kernel<3, true>) : go(add_rmsnorm_fp8_kernel<3, false>); break;
    default: res ? go(add_rmsnorm_fp8_kernel<4, true>) : go(add_rmsnorm_fp8_kernel<4, false>); break;
  }
  SG_LAUNCH_CHECK();
  return SG_OK;
}
