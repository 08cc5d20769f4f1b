// Products in e4m3 with fp32 scales: out = X W^T, X [R, K] with a scale for each
// row and 128 columns, W [N, K] with one for each 128 x 128 block.
//
//   out[r, c] = bf16( sum_b sx[b, r] * sw[c/128, b] * sum_{k in block b} x[r, k] w[c, k] )
//
// A block of 128 columns is exactly one v_mfma_f32_16x16x128 product, so its sum
// leaves the matrix pipe by itself, is scaled in fp32 and added to the
// accumulator.  The product is taken as W X^T: an output column of the MFMA (a
// lane's) is then an activation row, whose scale is one register a lane, and the
// weight's scale is one value for the wave: 4 fused multiply-adds for each
// product, and none of the scales ever needs spreading.
//
// The weight is packed once: 16-row x 128-column blocks of 2 KB in the order of
// the MFMA's operand (lane l: row l%16, columns 32 (l/16) .. +31 as two 16-byte
// pieces, piece j of all lanes together), so that copies and fragment reads are
// linear.  Blocks of 128 rows follow each other along K.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "sg_common.h"

namespace sg {
namespace {

typedef __attribute__((ext_vector_type(4))) float floatx4;
typedef __attribute__((ext_vector_type(8))) int intx8;

constexpr int kBlockK = 128;
constexpr int kPackRows = 128;                       // weight rows of a packed stripe
constexpr int kStripeBytes = kPackRows * kBlockK;    // a stripe's bytes per block of K
constexpr int kXcds = 8;

struct MatmulArgs {
  const unsigned char* x;
  int64_t x_stride;
  const float* x_scales;
  int64_t x_scale_stride;
  const unsigned char* w;
  const float* w_scales;
  uint16_t* out;
  int64_t out_stride;
  float* partial;  // [splits][R][padded N], nullptr when one workgroup takes all of K
  int rows, n, steps;  // steps: blocks of 128 columns
  int splits;
};

__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) char*)p));
}
// HBM -> LDS copies: lane i's 16 (4) bytes at gbase + voff land at lds + 16 i (4 i).
// The compiler does not see them; the kernel waits by s_waitcnt.
__device__ __forceinline__ void dma16(const void* gbase, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(lds), "v"(voff), "s"(gbase)
               : "memory", "m0");
}
__device__ __forceinline__ void dma4(const void* gbase, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2"
               :
               : "s"(lds), "v"(voff), "s"(gbase)
               : "memory", "m0");
}
constexpr int vmcnt_encoding(int n) {
  return (n & 15) | ((n >> 4) << 14) | (7 << 4) | (15 << 8);
}

__device__ __forceinline__ intx8 operand(uint4 lo, uint4 hi) {
  struct Two {
    uint4 a, b;
  };
  return __builtin_bit_cast(intx8, (Two{lo, hi}));
}

// BN x BM outputs (weight rows x activation rows) by WN x WM waves.
template <int BN, int BM, int WN, int WM, int STAGES>
struct Tile {
  static constexpr int kWaves = WN * WM;
  static constexpr int kThreads = 64 * kWaves;
  static constexpr int NB = BN / WN / 16;
  static constexpr int MB = BM / WM / 16;
  static constexpr int kWBytes = BN * kBlockK;
  static constexpr int kXBytes = BM * kBlockK;
  static constexpr int kScaleBytes = (BM + 63) / 64 * 256;
  static constexpr int kStage = kWBytes + kXBytes + kScaleBytes;
  static constexpr int kWCopies = kWBytes / 1024;
  static constexpr int kXCopies = kXBytes / 1024;
  static constexpr int kCopies = (kWCopies + kXCopies) / kWaves;  // per wave, + 1 of scales
  static_assert((kWCopies + kXCopies) % kWaves == 0, "copies spread evenly");
  static constexpr int kPitch = NB * 32 + 16;
  static constexpr int kStaging = kWaves * MB * 16 * kPitch;
  static constexpr int kLds = STAGES * kStage > kStaging ? STAGES * kStage : kStaging;
};

template <int BN, int BM, int WN, int WM, int STAGES, int PER_CU>
__global__ __launch_bounds__(64 * WN * WM, PER_CU * WN * WM / 4 < 1 ? 1 : PER_CU * WN * WM / 4)
    void fp8_matmul_kernel(MatmulArgs a, int n_tiles, int m_tiles) {
  using T = Tile<BN, BM, WN, WM, STAGES>;
  __shared__ __align__(1024) unsigned char smem[T::kLds];
  // Workgroup b runs on XCD b % 8: the row tiles of one weight tile take
  // consecutive slots of one XCD, whose L2 serves the weight to all of them.
  const int slot = blockIdx.x / kXcds;
  const int mt = slot % m_tiles;
  const int nt = (slot / m_tiles) * kXcds + blockIdx.x % kXcds;
  if (nt >= n_tiles) return;
  const int split = blockIdx.y;
  const int first = static_cast<int>(static_cast<int64_t>(a.steps) * split / a.splits);
  const int steps = static_cast<int>(static_cast<int64_t>(a.steps) * (split + 1) / a.splits) - first;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = nt * BN;
  const int m0 = mt * BM;
  const int wn = wave % WN;
  const int wm = wave / WN;

  // Copies of this wave: weight pieces are linear in the packed stripes, x rows
  // are 128 bytes whose 16-byte chunk c goes to LDS chunk c ^ (row & 7), so that
  // eight lanes reading one chunk of eight rows touch all banks.
  const unsigned char* wsrc[T::kCopies];
  uint32_t off[T::kCopies], dst[T::kCopies];
  bool is_w[T::kCopies];
#pragma unroll
  for (int i = 0; i < T::kCopies; ++i) {
    const int c = wave * T::kCopies + i;
    is_w[i] = c < T::kWCopies;
    dst[i] = 1024u * c;
    if (is_w[i]) {
      // 1 KB piece c of the tile's BN x 128 block: stripe c / 16, piece c % 16.
      wsrc[i] = a.w + (static_cast<int64_t>(n0 / kPackRows + c / 16) * a.steps + first) *
                          kStripeBytes + (n0 % kPackRows) * kBlockK + 1024 * (c % 16);
      off[i] = 16u * lane;
    } else {
      const int row = 8 * (c - T::kWCopies) + lane / 8;
      wsrc[i] = a.x + static_cast<int64_t>(m0) * a.x_stride + first * kBlockK;
      off[i] = static_cast<uint32_t>((min(m0 + row, a.rows - 1) - m0) * a.x_stride +
                                     16 * ((lane % 8) ^ (row & 7)));
    }
  }
  const int s_rows = 64 * (wave % ((BM + 63) / 64));
  const uint32_t s_off = 4u * (min(m0 + s_rows + lane, a.rows - 1) - m0);
  const unsigned char* s_src = reinterpret_cast<const unsigned char*>(
      a.x_scales + first * a.x_scale_stride + m0);
  const uint32_t ring = lds_addr(smem);
  auto issue = [&](int s) {
    const uint32_t stage = ring + (s % STAGES) * T::kStage;
#pragma unroll
    for (int i = 0; i < T::kCopies; ++i)
      dma16(wsrc[i] + static_cast<int64_t>(s) * (is_w[i] ? kStripeBytes : kBlockK), off[i],
            stage + dst[i]);
    dma4(s_src + 4 * static_cast<int64_t>(s) * a.x_scale_stride, s_off,
         stage + T::kWBytes + T::kXBytes + 4 * s_rows);
  };

  floatx4 acc[T::NB][T::MB];
#pragma unroll
  for (int i = 0; i < T::NB; ++i)
#pragma unroll
    for (int j = 0; j < T::MB; ++j) acc[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};

  const int q = lane >> 4;
  const int col = lane & 15;
  const int a_base = wn * T::NB * 2048 + 16 * lane;
  const int x_row = wm * T::MB * 16 + col;  // rows of further blocks share its low bits
  const int x_base = T::kWBytes + x_row * kBlockK;
  const int x_lo = 16 * ((2 * q) ^ (x_row & 7));
  const int x_hi = 16 * ((2 * q + 1) ^ (x_row & 7));
  const int s_base = T::kWBytes + T::kXBytes + 4 * x_row;
  // The constant address space makes these loads scalar: a vector load's wait
  // would drain the copies in flight.
  using ScalarFloat = const __attribute__((address_space(4))) float;
  ScalarFloat* w_scale = (ScalarFloat*)(
      a.w_scales + static_cast<int64_t>((n0 + wn * T::NB * 16) / kPackRows) * a.steps + first);

  for (int s = 0; s < STAGES - 1 && s < steps; ++s) issue(s);
  for (int s = 0; s < steps; ++s) {
    // Stage s has landed once only the copies of later stages are in flight.
    const int newer = min(STAGES - 2, steps - 1 - s);
    if (STAGES >= 4 && newer == 2) {
      __builtin_amdgcn_s_waitcnt(vmcnt_encoding(2 * (T::kCopies + 1)));
    } else if (STAGES >= 3 && newer >= 1) {
      __builtin_amdgcn_s_waitcnt(vmcnt_encoding(T::kCopies + 1));
    } else {
      __builtin_amdgcn_s_waitcnt(vmcnt_encoding(0));
    }
    __syncthreads();
    if (s + STAGES - 1 < steps) issue(s + STAGES - 1);
    const unsigned char* st = smem + (s % STAGES) * T::kStage;
    const float sw = w_scale[s];
    intx8 wf[T::NB];
#pragma unroll
    for (int i = 0; i < T::NB; ++i)
      wf[i] = operand(*reinterpret_cast<const uint4*>(st + a_base + 2048 * i),
                      *reinterpret_cast<const uint4*>(st + a_base + 2048 * i + 1024));
#pragma unroll
    for (int j = 0; j < T::MB; ++j) {
      const unsigned char* xr = st + x_base + 2048 * j;
      const intx8 xf = operand(*reinterpret_cast<const uint4*>(xr + x_lo),
                               *reinterpret_cast<const uint4*>(xr + x_hi));
      const float sc = *reinterpret_cast<const float*>(st + s_base + 64 * j) * sw;
#pragma unroll
      for (int i = 0; i < T::NB; ++i) {
        const floatx4 p = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
            wf[i], xf, floatx4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(p[e], sc, acc[i][j][e]);
      }
    }
  }

  // acc[i][j][e]: weight row n0 + wn 16 NB + 16 i + 4 q + e, activation row
  // m0 + wm 16 MB + 16 j + col.
  const int n_wave = n0 + wn * T::NB * 16;
  const int m_wave = m0 + wm * T::MB * 16;
  if (a.partial != nullptr) {
    const int64_t pitch = static_cast<int64_t>((a.n + kPackRows - 1) / kPackRows) * kPackRows;
#pragma unroll
    for (int j = 0; j < T::MB; ++j) {
      const int row = m_wave + 16 * j + col;
      if (row >= a.rows) continue;
      float* p = a.partial + (static_cast<int64_t>(split) * a.rows + row) * pitch + n_wave + 4 * q;
#pragma unroll
      for (int i = 0; i < T::NB; ++i) *reinterpret_cast<floatx4*>(p + 16 * i) = acc[i][j];
    }
    return;
  }
  __syncthreads();  // the ring becomes the staging area of whole output rows
  unsigned char* stage = smem + wave * T::MB * 16 * T::kPitch;
#pragma unroll
  for (int j = 0; j < T::MB; ++j)
#pragma unroll
    for (int i = 0; i < T::NB; ++i)
      *reinterpret_cast<uint2*>(stage + (16 * j + col) * T::kPitch + 2 * (16 * i + 4 * q)) =
          make_uint2(pack_bf16x2(acc[i][j][0], acc[i][j][1]),
                     pack_bf16x2(acc[i][j][2], acc[i][j][3]));
  __builtin_amdgcn_wave_barrier();
  constexpr int kLanes = T::NB * 2;  // 16-byte chunks of a row
  for (int k = lane; k < T::MB * 16 * kLanes; k += 64) {
    const int r = k / kLanes;
    const int c = k % kLanes;
    const int row = m_wave + r;
    const int n = n_wave + 8 * c;
    if (row >= a.rows || n >= a.n) continue;
    const uint4 v = *reinterpret_cast<const uint4*>(stage + r * T::kPitch + 16 * c);
    uint16_t* dst_row = a.out + row * a.out_stride + n;
    if (n + 8 <= a.n) {
      *reinterpret_cast<uint4*>(dst_row) = v;
    } else {
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      for (int e = 0; n + e < a.n; ++e)
        dst_row[e] = static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1)));
    }
  }
}

// Adds the splits' partial sums in their order; eight columns a thread.
__global__ __launch_bounds__(256) void fp8_matmul_join_kernel(MatmulArgs a, int chunks) {
  const int64_t item = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x;
  const int64_t row = item / chunks;
  if (row >= a.rows) return;
  const int n = 8 * static_cast<int>(item - row * chunks);
  const int64_t pitch = static_cast<int64_t>((a.n + kPackRows - 1) / kPackRows) * kPackRows;
  float s[8] = {};
  for (int k = 0; k < a.splits; ++k) {
    const float4* p = reinterpret_cast<const float4*>(
        a.partial + (static_cast<int64_t>(k) * a.rows + row) * pitch + n);
    const float4 lo = p[0], hi = p[1];
    s[0] += lo.x; s[1] += lo.y; s[2] += lo.z; s[3] += lo.w;
    s[4] += hi.x; s[5] += hi.y; s[6] += hi.z; s[7] += hi.w;
  }
  uint16_t* dst = a.out + row * a.out_stride + n;
  if (n + 8 <= a.n) {
    *reinterpret_cast<uint4*>(dst) =
        make_uint4(pack_bf16x2(s[0], s[1]), pack_bf16x2(s[2], s[3]), pack_bf16x2(s[4], s[5]),
                   pack_bf16x2(s[6], s[7]));
  } else {
    for (int e = 0; n + e < a.n; ++e) dst[e] = f32_to_bf16(s[e]);
  }
}

// 16 bytes a thread of the packed weight.
__global__ __launch_bounds__(256) void fp8_pack_kernel(const unsigned char* __restrict__ w,
                                                       int64_t stride, int n, int k, int steps,
                                                       uint4* __restrict__ out, int64_t total) {
  const int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x;
  if (i >= total) return;
  const int lane = static_cast<int>(i & 63);
  const int piece = static_cast<int>(i >> 6) & 1;
  const int blk = static_cast<int>(i >> 7) & 7;
  const int64_t cell = i >> 10;
  const int64_t row = cell / steps * kPackRows + 16 * blk + (lane & 15);
  const int64_t col = cell % steps * kBlockK + 32 * (lane >> 4) + 16 * piece;
  unsigned char b[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) b[e] = row < n && col + e < k ? w[row * stride + col + e] : 0;
  uint4 v;
  __builtin_memcpy(&v, b, 16);
  out[i] = v;
}

// How a call is cut.
struct Cut {
  int bm;      // activation rows of a tile
  int splits;  // of K
};

Cut cut_of(int rows, int n, int steps) {
  Cut c;
  c.bm = rows <= 32 ? 32 : rows <= 64 ? 64 : 128;
  const int64_t tiles = static_cast<int64_t>((n + 127) / 128) * ((rows + c.bm - 1) / c.bm);
  c.splits = 1;
  if (tiles < 384) {
    const int64_t want = (512 + tiles - 1) / tiles;
    c.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(want, steps / 4)));
  }
  return c;
}

bool sizes_ok(int32_t rows, int32_t n, int32_t k) {
  return rows >= 0 && n >= 1 && n <= (1 << 24) && k >= 1 && k <= (1 << 24);
}

}  // namespace
}  // namespace sg

extern "C" int64_t sg_fp8_packed_bytes(int32_t n, int32_t k) {
  if (!sg::sizes_ok(0, n, k)) return -1;
  return static_cast<int64_t>((n + 127) / 128 * 128) * ((k + 127) / 128 * 128);
}

extern "C" int sg_fp8_pack_weight(const void* weight_dev, int64_t weight_row_stride, int32_t n,
                                  int32_t k, void* packed_dev, sg_stream_t stream) {
  using namespace sg;
  clear_error();
  SG_REQUIRE(sizes_ok(0, n, k), "n and k must lie in [1, 2^24]");
  SG_REQUIRE(weight_dev && packed_dev, "null device pointer");
  SG_REQUIRE(weight_row_stride >= k, "weight_row_stride must cover a row");
  SG_REQUIRE((reinterpret_cast<uintptr_t>(packed_dev) & 15) == 0,
             "packed_dev must be 16-byte aligned");
  const int64_t total = sg_fp8_packed_bytes(n, k) / 16;
  SG_REQUIRE((total + 255) / 256 <= INT_MAX, "weight too large");
  fp8_pack_kernel<<<dim3(static_cast<unsigned>((total + 255) / 256)), dim3(256), 0,
                    static_cast<hipStream_t>(stream)>>>(
      static_cast<const unsigned char*>(weight_dev), weight_row_stride, n, k, (k + 127) / 128,
      static_cast<uint4*>(packed_dev), total);
  SG_LAUNCH_CHECK();
  return SG_OK;
}

extern "C" int64_t sg_fp8_matmul_workspace_bytes(int32_t num_rows, int32_t n, int32_t k) {
  using namespace sg;
  if (!sizes_ok(num_rows, n, k)) return -1;
  if (num_rows == 0) return 0;
  const Cut c = cut_of(num_rows, n, (k + 127) / 128);
  return c.splits == 1 ? 0
                       : static_cast<int64_t>(c.splits) * num_rows * ((n + 127) / 128 * 128) * 4;
}

extern "C" int sg_fp8_matmul(const SgFp8MatmulArgs* args, sg_stream_t stream) {
  using namespace sg;
  clear_error();
  SG_REQUIRE(args != nullptr, "null SgFp8MatmulArgs");
  const SgFp8MatmulArgs& a = *args;
  SG_REQUIRE(sizes_ok(a.num_rows, a.n, a.k), "rows must not be negative, n and k in [1, 2^24]");
  if (a.num_rows == 0) return SG_OK;
  const int steps = (a.k + 127) / 128;
  SG_REQUIRE(a.codes_dev && a.scales_dev && a.weight_dev && a.weight_scales_dev && a.out_dev,
             "null device pointer");
  SG_REQUIRE(a.code_stride >= static_cast<int64_t>(steps) * 128 && a.code_stride % 16 == 0 &&
                 a.code_stride < (int64_t{1} << 25),
             "code_stride must be a multiple of 16 in [K padded to 128, 2^25)");
  SG_REQUIRE(a.scale_stride >= a.num_rows, "scale_stride must cover the rows");
  SG_REQUIRE(a.out_stride >= a.n && a.out_stride % 8 == 0,
             "out_stride must cover a row and be a multiple of 8");
  SG_REQUIRE(((reinterpret_cast<uintptr_t>(a.codes_dev) |
               reinterpret_cast<uintptr_t>(a.weight_dev) |
               reinterpret_cast<uintptr_t>(a.out_dev)) & 15) == 0 &&
                 ((reinterpret_cast<uintptr_t>(a.scales_dev) |
                   reinterpret_cast<uintptr_t>(a.weight_scales_dev)) & 3) == 0,
             "codes, the packed weight and out must be 16-byte aligned");
  const Cut c = cut_of(a.num_rows, a.n, steps);
  const int64_t need = sg_fp8_matmul_workspace_bytes(a.num_rows, a.n, a.k);
  SG_REQUIRE(need == 0 || (a.workspace_dev && a.workspace_bytes >= static_cast<size_t>(need) &&
                           (reinterpret_cast<uintptr_t>(a.workspace_dev) & 15) == 0),
             "workspace below sg_fp8_matmul_workspace_bytes");
  MatmulArgs m;
  m.x = static_cast<const unsigned char*>(a.codes_dev);
  m.x_stride = a.code_stride;
  m.x_scales = a.scales_dev;
  m.x_scale_stride = a.scale_stride;
  m.w = static_cast<const unsigned char*>(a.weight_dev);
  m.w_scales = a.weight_scales_dev;
  m.out = static_cast<uint16_t*>(a.out_dev);
  m.out_stride = a.out_stride;
  m.partial = c.splits > 1 ? static_cast<float*>(a.workspace_dev) : nullptr;
  m.rows = a.num_rows;
  m.n = a.n;
  m.steps = steps;
  m.splits = c.splits;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  auto go = [&](auto kernel, int bn, int bm, int threads) {
    const int n_tiles = (a.n + bn - 1) / bn;
    const int m_tiles = (a.num_rows + bm - 1) / bm;
    const int64_t blocks = static_cast<int64_t>((n_tiles + kXcds - 1) / kXcds * kXcds) * m_tiles;
    if (blocks > INT_MAX) return false;
    kernel<<<dim3(static_cast<unsigned>(blocks), c.splits), dim3(threads), 0, s>>>(m, n_tiles,
                                                                                    m_tiles);
    return true;
  };
  bool launched;
  switch (c.bm) {
    case 32: launched = go(fp8_matmul_kernel<128, 32, 4, 1, 3, 2>, 128, 32, 256); break;
    case 64: launched = go(fp8_matmul_kernel<128, 64, 2, 2, 3, 2>, 128, 64, 256); break;
    default: launched = go(fp8_matmul_kernel<128, 128, 2, 2, 2, 2>, 128, 128, 256); break;
  }
  SG_REQUIRE(launched, "too many tiles");
  SG_LAUNCH_CHECK();
  if (c.splits > 1) {
    const int chunks = (a.n + 7) / 8;
    const int64_t items = static_cast<int64_t>(a.num_rows) * chunks;
    SG_REQUIRE((items + 255) / 256 <= INT_MAX, "too many outputs");
    fp8_matmul_join_kernel<<<dim3(static_cast<unsigned>((items + 255) / 256)), dim3(256), 0, s>>>(
        m, chunks);
    SG_LAUNCH_CHECK();
  }
  return SG_OK;
}
