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
// The instruction adds the products of 8 columns at a time, cut towards 0 to multiples
// of 2^(e - 13), e the largest sum of a column's two exponents; the 8-sums are added in
// fp32 (bit for bit so over a whole call).  7 products of 8 can lose, so a block's sum
// is off by less than 2^-10 of sum |x w| where one of every 8 products is some hundred
// times the others, by 2^-16.3 of it at most and 2^-19.5 in the mean over Gaussian rows.
// The e4m3 values themselves stand for rows and weights to 2^-4.
//
// The weight is packed once: 16-row x 128-column blocks of 2 KB in the order of
// the MFMA's operand (lane l: row l%16, columns 64 j + 16 (l/16) .. +15 as 16-byte
// piece j of two, a piece of all lanes together), so that copies and fragment reads
// are linear.  (Which 32 columns a lane group multiplies does not matter as long as
// both operands agree.)  Blocks of 128 rows follow each other along K.
#include <algorithm>
#include <climits>
#include <cmath>
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

// Activations in LDS: two halves of 64 columns, rows of 64 bytes whose 16-byte
// chunk c is at c ^ ((row >> 1) & 3); a fragment read (lane l: row l%16, chunk l/16)
// then has no bank conflicts (rows of 128 bytes with chunk c at c ^ (row & 7): 4.75
// conflict cycles a read).  Offset from row m0 that this lane copies in 1 KB piece
// c of a tile of bm rows: 16 rows, four lanes a row.  Rows past the last re-read it.
__device__ __forceinline__ uint32_t x_piece(const MatmulArgs& a, int m0, int bm, int c, int lane) {
  const int half = c / (bm / 16);
  const int row = 16 * (c - half * (bm / 16)) + lane / 4;
  return static_cast<uint32_t>((min(m0 + row, a.rows - 1) - m0) * a.x_stride + 64 * half +
                               16 * ((lane & 3) ^ ((row >> 1) & 3)));
}

// Eight output columns from n on of a row, as far as they exist.
__device__ __forceinline__ void store_chunk(const MatmulArgs& a, int row, int n, uint4 v) {
  if (row >= a.rows || n >= a.n) return;
  uint16_t* dst = a.out + row * a.out_stride + n;
  if (n + 8 <= a.n) {
    *reinterpret_cast<uint4*>(dst) = v;
  } else {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    for (int e = 0; n + e < a.n; ++e) dst[e] = static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1)));
  }
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
  static_assert(STAGES >= 2 && STAGES <= 6 && (STAGES - 2) * (kCopies + 1) < 64,
                "waits count at most 63 copies");
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

  // Copies of this wave: weight pieces are linear in the packed stripes; for x see
  // x_piece.
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
      wsrc[i] = a.x + static_cast<int64_t>(m0) * a.x_stride + first * kBlockK;
      off[i] = x_piece(a, m0, BM, c - T::kWCopies, lane);
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
  const int x_base = T::kWBytes + x_row * 64 + 16 * (q ^ ((x_row >> 1) & 3));
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
    if (newer == STAGES - 2) {
      __builtin_amdgcn_s_waitcnt(vmcnt_encoding((STAGES - 2) * (T::kCopies + 1)));
    } else {
      switch (newer) {
        case 4: __builtin_amdgcn_s_waitcnt(vmcnt_encoding(4 * (T::kCopies + 1))); break;
        case 3: __builtin_amdgcn_s_waitcnt(vmcnt_encoding(3 * (T::kCopies + 1))); break;
        case 2: __builtin_amdgcn_s_waitcnt(vmcnt_encoding(2 * (T::kCopies + 1))); break;
        case 1: __builtin_amdgcn_s_waitcnt(vmcnt_encoding(T::kCopies + 1)); break;
        default: __builtin_amdgcn_s_waitcnt(vmcnt_encoding(0)); break;
      }
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
      const unsigned char* xr = st + x_base + 1024 * j;
      const intx8 xf = operand(*reinterpret_cast<const uint4*>(xr),
                               *reinterpret_cast<const uint4*>(xr + 64 * BM));
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
    store_chunk(a, m_wave + r, n_wave + 8 * c,
                *reinterpret_cast<const uint4*>(stage + r * T::kPitch + 16 * c));
  }
}

// Ping-pong form: eight waves, two per SIMD, in two groups (waves 0-3 and 4-7) that
// alternate between reading a stage's fragments from LDS and multiplying, so that
// the matrix pipe of a SIMD works for one of its waves while the LDS serves the
// other.  Tile of 256 weight rows x 64 MB activation rows; wave w owns weight rows
// 128 (w & 1) .. +128 and activation rows 16 MB (w / 2) .. +16 MB.
//   phase 2t    group A reads stage t, group B multiplies stage t-1;
//   phase 2t+1  group B reads stage t, group A multiplies stage t.
// One barrier a phase.  Both groups issue stage t+1's copies in phase 2t, when the
// last reads of stage t-1 (its place in the two-stage ring) are over, and wait for
// them at the end of phase 2t+1.  A phase's products take 256 MB matrix cycles on
// each SIMD beside 512 + 128 MB cycles of fragment reads and 128 + 32 MB of copies.
template <int MB>
struct PpTile {
  static constexpr int BN = 256;
  static constexpr int BM = 64 * MB;
  static constexpr int kWBytes = BN * kBlockK;
  static constexpr int kXBytes = BM * kBlockK;
  static constexpr int kStage = kWBytes + kXBytes + 1024;
  static constexpr int kPitch = 8 * 32 + 16;
  static constexpr int kStaging = 8 * 16 * kPitch;  // one 16-row block a wave
};

template <int MB>
__global__ __launch_bounds__(512, 2) void fp8_matmul_pp_kernel(MatmulArgs a, int n_tiles,
                                                                int m_tiles) {
  using T = PpTile<MB>;
  constexpr int kLds = 2 * T::kStage > T::kStaging ? 2 * T::kStage : T::kStaging;
  __shared__ __align__(1024) unsigned char smem[kLds];
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
  const int wn = wave & 1;
  const int wm = wave >> 1;
  const int n0 = nt * T::BN;
  const int m0 = mt * T::BM;

  // Copies: wave w's four of the weight (half a stripe's 1 KB pieces 4 (w % 4) ..,
  // stripe w / 4), MB of the activations (8 rows each), one of 64 scales.  The
  // second stripe of a last odd tile re-reads the first.
  const int stripe = min(n0 / kPackRows + (wave >> 2), (a.n + kPackRows - 1) / kPackRows - 1);
  const unsigned char* w_src =
      a.w + (static_cast<int64_t>(stripe) * a.steps + first) * kStripeBytes + 4096 * (wave & 3);
  const uint32_t w_off = 16u * lane;
  const unsigned char* x_src = a.x + static_cast<int64_t>(m0) * a.x_stride + first * kBlockK;
  uint32_t x_off[MB];
#pragma unroll
  for (int i = 0; i < MB; ++i) x_off[i] = x_piece(a, m0, T::BM, wave * MB + i, lane);
  const int s_rows = 64 * ((wave & 3) % MB);
  const uint32_t s_off = 4u * (min(m0 + s_rows + lane, a.rows - 1) - m0);
  const unsigned char* s_src = reinterpret_cast<const unsigned char*>(
      a.x_scales + first * a.x_scale_stride + m0);
  const uint32_t ring = lds_addr(smem);
  auto issue = [&](int s) {
    const uint32_t stage = ring + (s & 1) * T::kStage;
    const unsigned char* ws = w_src + static_cast<int64_t>(s) * kStripeBytes;
#pragma unroll
    for (int i = 0; i < 4; ++i) dma16(ws + 1024 * i, w_off, stage + 4096u * wave + 1024u * i);
    const unsigned char* xs = x_src + static_cast<int64_t>(s) * kBlockK;
#pragma unroll
    for (int i = 0; i < MB; ++i)
      dma16(xs, x_off[i], stage + T::kWBytes + 1024u * (wave * MB + i));
    dma4(s_src + 4 * static_cast<int64_t>(s) * a.x_scale_stride, s_off,
         stage + T::kWBytes + T::kXBytes + 4 * s_rows);
  };
  constexpr int kCopies = 4 + MB + 1;

  floatx4 acc[8][MB];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < MB; ++j) acc[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  const int q = lane >> 4;
  const int col = lane & 15;
  const int a_base = wn * 16384 + 16 * lane;
  const int x_row = wm * MB * 16 + col;
  const int x_base = T::kWBytes + x_row * 64 + 16 * (q ^ ((x_row >> 1) & 3));
  const int s_base = T::kWBytes + T::kXBytes + 4 * x_row;
  using ScalarFloat = const __attribute__((address_space(4))) float;
  const int w_block = min((n0 + 128 * wn) / kPackRows, (a.n + kPackRows - 1) / kPackRows - 1);
  ScalarFloat* w_scale =
      (ScalarFloat*)(a.w_scales + static_cast<int64_t>(w_block) * a.steps + first);

  auto body = [&](auto group) {
    constexpr int G = decltype(group)::value;
    intx8 wf[8], xf[MB];
    float sc[MB];
    auto read = [&](int s) {
      const unsigned char* st = smem + (s & 1) * T::kStage;
      const float sw = w_scale[s];
#pragma unroll
      for (int j = 0; j < MB; ++j) {
        const unsigned char* xr = st + x_base + 1024 * j;
        xf[j] = operand(*reinterpret_cast<const uint4*>(xr),
                        *reinterpret_cast<const uint4*>(xr + 64 * T::BM));
        sc[j] = *reinterpret_cast<const float*>(st + s_base + 64 * j) * sw;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        wf[i] = operand(*reinterpret_cast<const uint4*>(st + a_base + 2048 * i),
                        *reinterpret_cast<const uint4*>(st + a_base + 2048 * i + 1024));
    };
    // Product k = 8 j + i; the scaled addition of a product follows two later.
    auto multiply = [&]() {
      floatx4 p[3];
      constexpr int kAll = 8 * MB;
#pragma unroll
      for (int k = 0; k < kAll + 2; ++k) {
        if (k < kAll)
          p[k % 3] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
              wf[k % 8], xf[k / 8], floatx4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0, 0, 0, 0);
        if (k >= 2) {
          const int d = k - 2;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            acc[d % 8][d / 8][e] = __builtin_fmaf(p[d % 3][e], sc[d / 8], acc[d % 8][d / 8][e]);
        }
        // In this order: a product's result is not waited for.
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    // The fences keep reads and products inside their phases.
    auto end_phase = [&](bool landed) {
      if (landed) __builtin_amdgcn_s_waitcnt(0xf70);  // vmcnt(0): stage t+1's copies
      __builtin_amdgcn_s_waitcnt(0xc07f);             // lgkmcnt(0): this phase's reads
      __builtin_amdgcn_sched_barrier(0);
      __syncthreads();
      __builtin_amdgcn_sched_barrier(0);
    };
    issue(0);
    if (steps > 1) issue(1);
    if (steps > 1) {
      __builtin_amdgcn_s_waitcnt(vmcnt_encoding(kCopies));
    } else {
      __builtin_amdgcn_s_waitcnt(vmcnt_encoding(0));
    }
    __syncthreads();
    if constexpr (G == 1) end_phase(false);  // phase 0: group A reads stage 0
    for (int t = 0; t < steps; ++t) {
      read(t);
      if (G == 0 && t > 0 && t + 1 < steps) issue(t + 1);
      end_phase(G == 1);
      if (G == 1 && t + 2 < steps) issue(t + 2);
      multiply();
      end_phase(G == 0);
    }
    if constexpr (G == 0) end_phase(false);  // group B's last products
  };
  if (wave < 4) {
    body(std::integral_constant<int, 0>{});
  } else {
    body(std::integral_constant<int, 1>{});
  }

  const int n_wave = n0 + 128 * wn;
  const int m_wave = m0 + wm * MB * 16;
  if (a.partial != nullptr) {
    const int64_t pitch = static_cast<int64_t>((a.n + kPackRows - 1) / kPackRows) * kPackRows;
    if (n_wave >= pitch) return;
#pragma unroll
    for (int j = 0; j < MB; ++j) {
      const int row = m_wave + 16 * j + col;
      if (row >= a.rows) continue;
      float* p = a.partial + (static_cast<int64_t>(split) * a.rows + row) * pitch + n_wave + 4 * q;
#pragma unroll
      for (int i = 0; i < 8; ++i) *reinterpret_cast<floatx4*>(p + 16 * i) = acc[i][j];
    }
    return;
  }
  unsigned char* stage = smem + wave * 16 * T::kPitch;
#pragma unroll
  for (int j = 0; j < MB; ++j) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      *reinterpret_cast<uint2*>(stage + col * T::kPitch + 2 * (16 * i + 4 * q)) =
          make_uint2(pack_bf16x2(acc[i][j][0], acc[i][j][1]),
                     pack_bf16x2(acc[i][j][2], acc[i][j][3]));
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = m_wave + 16 * j + 4 * r + (lane >> 4);
      const int n = n_wave + 8 * (lane & 15);
      const uint4 v = *reinterpret_cast<const uint4*>(stage + (4 * r + (lane >> 4)) * T::kPitch +
                                                      16 * (lane & 15));
      store_chunk(a, row, n, v);
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// Few activation rows: bound by the weight's bytes.  A wave multiplies 16 NB weight
// rows by 16 MB activation rows over its share of K, both operands loaded straight
// into registers (a weight byte is used by one wave only, so LDS would add a copy
// and a barrier); the KW waves of a workgroup take turns over the blocks of K and
// their sums are added in LDS, in the order of the waves: one launch, no workspace.
// Blocks are loaded kAhead at a time while the last ones are multiplied.
template <int NB, int MB, int KW>
__global__ __launch_bounds__(64 * KW) void fp8_matmul_few_kernel(MatmulArgs a) {
  constexpr int kAhead = NB * MB >= 4 ? 1 : 2;
  constexpr int kSums = 4 * NB * MB;  // accumulators of a lane
  __shared__ float s_sum[KW > 1 ? (KW - 1) * kSums * 64 : 1];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int q = lane >> 4;
  const int col = lane & 15;
  const int n0 = blockIdx.x * 16 * NB;
  const int m0 = blockIdx.y * 16 * MB;
  const unsigned char* w = a.w + static_cast<int64_t>(n0 / kPackRows) * a.steps * kStripeBytes +
                           n0 % kPackRows * kBlockK;
  const unsigned char* x = a.x + static_cast<int64_t>(m0) * a.x_stride;
  const float* xs = a.x_scales + m0;
  uint32_t x_off[MB], s_off[MB];
#pragma unroll
  for (int j = 0; j < MB; ++j) {
    const int row = min(m0 + 16 * j + col, a.rows - 1) - m0;  // past the end: the last row
    x_off[j] = static_cast<uint32_t>(row * a.x_stride) + 16 * q;
    s_off[j] = row;
  }
  using ScalarFloat = const __attribute__((address_space(4))) float;
  ScalarFloat* w_scale =
      (ScalarFloat*)(a.w_scales + static_cast<int64_t>(n0 / kPackRows) * a.steps);
  struct Step {
    uint4 w[NB][2], x[MB][2];
    float xs[MB], ws;
  };
  auto load = [&](int s, Step& t) {
    const unsigned char* wb = w + static_cast<int64_t>(s) * kStripeBytes;
    const unsigned char* xb = x + static_cast<int64_t>(s) * kBlockK;
    const float* sb = xs + static_cast<int64_t>(s) * a.x_scale_stride;
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int p = 0; p < 2; ++p)
        t.w[i][p] = *reinterpret_cast<const uint4*>(wb + 2048 * i + 1024 * p + 16 * lane);
#pragma unroll
    for (int j = 0; j < MB; ++j) {
#pragma unroll
      for (int p = 0; p < 2; ++p)
        t.x[j][p] = *reinterpret_cast<const uint4*>(xb + x_off[j] + 64 * p);
      t.xs[j] = sb[s_off[j]];
    }
    t.ws = w_scale[s];
  };
  floatx4 acc[NB][MB];
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < MB; ++j) acc[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  auto multiply = [&](const Step& t) {
#pragma unroll
    for (int j = 0; j < MB; ++j) {
      const float sc = t.xs[j] * t.ws;
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const floatx4 p = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
            operand(t.w[i][0], t.w[i][1]), operand(t.x[j][0], t.x[j][1]),
            floatx4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(p[e], sc, acc[i][j][e]);
      }
    }
  };
  // This wave's blocks are wave, wave + KW, ...
  const int mine = a.steps > wave ? (a.steps - wave + KW - 1) / KW : 0;
  auto block = [&](int k) { return wave + KW * k; };
  // Two sets of kAhead blocks take turns.  (One set copied into the other at the end of
  // a turn made every turn wait for the loads it had issued.)
  Step set[2][kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; ++u)
    if (u < mine) load(block(u), set[0][u]);
  int k = 0;
  auto turn = [&](auto parity) {  // of the blocks k .. in set[parity]
    constexpr int p = decltype(parity)::value;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) load(block(k + kAhead + u), set[1 - p][u]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) multiply(set[p][u]);
    k += kAhead;
  };
  auto finish = [&](Step (&last)[kAhead]) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (k + u < mine) multiply(last[u]);
    for (k += kAhead; k < mine; ++k) {
      load(block(k), last[0]);
      multiply(last[0]);
    }
  };
  using Even = std::integral_constant<int, 0>;
  using Odd = std::integral_constant<int, 1>;
  while (k + 3 * kAhead <= mine) {
    turn(Even{});
    turn(Odd{});
  }
  if (k + 2 * kAhead <= mine) {
    turn(Even{});
    finish(set[1]);
  } else {
    finish(set[0]);
  }

  if (KW > 1) {
    if (wave > 0) {
      float* d = s_sum + (wave - 1) * kSums * 64 + lane;
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int j = 0; j < MB; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) d[64 * (4 * (i * MB + j) + e)] = acc[i][j][e];
    }
    __syncthreads();
    if (wave > 0) return;
    for (int v = 0; v < KW - 1; ++v) {
      const float* d = s_sum + v * kSums * 64 + lane;
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int j = 0; j < MB; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] += d[64 * (4 * (i * MB + j) + e)];
    }
  }
#pragma unroll
  for (int j = 0; j < MB; ++j) {
    const int row = m0 + 16 * j + col;
    if (row >= a.rows) continue;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int n = n0 + 16 * i + 4 * q;
      uint16_t* dst = a.out + row * a.out_stride + n;
      const uint32_t v[2] = {pack_bf16x2(acc[i][j][0], acc[i][j][1]),
                             pack_bf16x2(acc[i][j][2], acc[i][j][3])};
      if (n + 4 <= a.n) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(v[0], v[1]);
      } else {
        for (int e = 0; e < 4 && n + e < a.n; ++e)
          dst[e] = static_cast<uint16_t>(v[e >> 1] >> (16 * (e & 1)));
      }
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
  const int64_t col = cell % steps * kBlockK + 64 * piece + 16 * (lane >> 4);
  unsigned char b[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) b[e] = row < n && col + e < k ? w[row * stride + col + e] : 0;
  uint4 v;
  __builtin_memcpy(&v, b, 16);
  out[i] = v;
}

// How a call is cut: a kernel and the splits of K.
enum Form { kFew1, kFew2, kFew1x2, kFew2x2, kTile64, kTile64Pair, kTile128, kTile128Pair, kPp3, kPp4 };
struct Cut {
  Form form;
  int splits;
};

// Rows up to 32 take the few-rows kernel; 33 to 64, which read the weight twice there,
// while it has at most 48 MiB (N x K).  Few-rows and tile kernels at 64 rows, a launch's
// share of many with weights from HBM: 2560 -> 6144 in 9.8 and 13.6 us, 4096 -> 4096 9.0
// and 15.3, 4096 -> 12288 20.8 and 18.9, 12288 -> 4096 19.5 and 19.0; 12288 -> 6144 34.7
// and 26.9, 4096 -> 16384 26.4 and 21.2, 4096 -> 24576 38.6 and 24.6 (33 rows: 8.2 and
// 11.5, 8.4 and 13.2, 18.7 and 18.9, 17.9 and 17.8; 28.2 and 24.5, 24.8 and 20.1, 36.3
// and 22.7).  Whether a weight block's two readers share an XCD makes no difference
// (4096 -> 6144, where they do, 14.0; 6176, where they do not, 14.1).  Two weight blocks a
// wave once that leaves 160 workgroups (6144 x 2560 at 16 rows 4.4 us, one block 5.2;
// at 32 rows 7.7 and 9.4; 4096 x 12288 the other way round, 10.8 and 9.4, at 32 rows
// 21.2 and 18.5).
//
// Beyond, the tile kernels by an estimate: rounds of workgroups x blocks of K x
// the time of a block (us, measured with every CU at work on 4096 -> 24576 and
// 12288 -> 4096, each pass with another weight, so that weights come from HBM), and
// for splits the partial sums' way through memory and back.  Measured against each
// other (us, the best and the next form): 2,048 rows of 4096 -> 24576 ping-pong 187,
// 128 x 128 pairs 234; of 12288 -> 4096 ping-pong in two splits 109, pairs 111; of
// 4096 -> 4096 pairs 42, ping-pong 54; 128 rows of 4096 -> 24576 one 128-row tile a
// CU 29, pairs 38; 512 rows of 2560 -> 6144 the same 18, 64-row pairs 22; 512 of
// 4096 -> 4096 64-row pairs 21, 128-row tiles 24; 256 of it one 64-row tile a CU 19,
// pairs 20.
Cut cut_of(int rows, int n, int steps) {
  if (rows <= 16) return {n > 32 * 159 ? kFew2 : kFew1, 1};
  const int64_t weight_bytes = static_cast<int64_t>(n) * steps * kBlockK;
  if (rows <= 32 || (rows <= 64 && weight_bytes <= (48 << 20)))
    return {(n + 31) / 32 * ((rows + 31) / 32) < 160 ? kFew1x2 : kFew2x2, 1};
  struct Kind {
    Form form;
    int bn, bm, slots;  // workgroups at a time
    double block_us;
  };
  static const Kind kinds[] = {{kTile64, 128, 64, 256, 0.55},  {kTile64Pair, 128, 64, 512, 0.90},
                               {kTile128, 128, 128, 256, 0.75}, {kTile128Pair, 128, 128, 512, 1.20},
                               {kPp3, 256, 192, 256, 1.45},     {kPp4, 256, 256, 256, 1.85}};
  Cut best = {kTile128Pair, 1};
  double least = 1e300;
  for (const Kind& k : kinds) {
    const double tiles = static_cast<double>((n + k.bn - 1) / k.bn) * ((rows + k.bm - 1) / k.bm);
    for (int splits : {1, 2, 3, 4, 6, 8}) {
      if (splits > 1 && steps < 4 * splits) break;
      const int per = (steps + splits - 1) / splits;
      double us = std::ceil(tiles * splits / k.slots) * per * k.block_us;
      if (splits > 1) us += 4.0 + splits * 8.0 * rows * n / 6e6;
      if (us < least) least = us, best = {k.form, splits};
    }
  }
  return best;
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

extern "C" int32_t sg_fp8_matmul_form(int32_t num_rows, int32_t n, int32_t k) {
  using namespace sg;
  if (!sizes_ok(num_rows, n, k) || num_rows == 0) return -1;
  const Cut c = cut_of(num_rows, n, (k + 127) / 128);
  return static_cast<int32_t>(c.form) + 16 * c.splits;
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
                 a.code_stride <= (int64_t{1} << 24),  // 255 rows on: 32-bit offsets
             "code_stride must be a multiple of 16 in [K padded to 128, 2^24]");
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
  auto few = [&](auto kernel, int nb, int mb) {
    kernel<<<dim3((a.n + 16 * nb - 1) / (16 * nb), (a.num_rows + 16 * mb - 1) / (16 * mb)),
             dim3(512), 0, s>>>(m);
    return true;
  };
  bool launched = false;
  switch (c.form) {
    case kFew1: launched = few(fp8_matmul_few_kernel<1, 1, 8>, 1, 1); break;
    case kFew2: launched = few(fp8_matmul_few_kernel<2, 1, 8>, 2, 1); break;
    case kFew1x2: launched = few(fp8_matmul_few_kernel<1, 2, 8>, 1, 2); break;
    case kFew2x2: launched = few(fp8_matmul_few_kernel<2, 2, 8>, 2, 2); break;
    case kTile64: launched = go(fp8_matmul_kernel<128, 64, 2, 4, 6, 1>, 128, 64, 512); break;
    case kTile64Pair: launched = go(fp8_matmul_kernel<128, 64, 2, 2, 3, 2>, 128, 64, 256); break;
    case kTile128: launched = go(fp8_matmul_kernel<128, 128, 2, 4, 4, 1>, 128, 128, 512); break;
    case kTile128Pair: launched = go(fp8_matmul_kernel<128, 128, 2, 2, 2, 2>, 128, 128, 256); break;
    case kPp3: launched = go(fp8_matmul_pp_kernel<3>, 256, 192, 512); break;
    case kPp4: launched = go(fp8_matmul_pp_kernel<4>, 256, 256, 512); break;
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
