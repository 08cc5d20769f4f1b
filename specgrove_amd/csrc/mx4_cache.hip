// The cache in 4 bits: packing the kept rows into the arena, and unpacking.
//
// A row's block of 32 values with largest magnitude A gets the scale 2^e, e the
// least integer with A <= 7 * 2^e; a value v is held as the e2m1 number nearest
// v / 2^e (grid 0, 1/2, 1, 3/2, 2, 3, 4, 6; 7 is where 6 and the next step, 8,
// meet).  With A = 1.m * 2^E in fp32 bits, A <= 1.75 * 2^(e+2) makes
// e = E - 2 + (1.m > 1.75): one integer add with carry into the exponent.
// gfx950 converts in both directions by itself (two values an instruction, the
// scale an operand; to nearest, ties to even).
//
// Both kernels are bound by HBM.  kv_commit_mx4_kernel reads 16 bytes (8 values)
// a lane; four lanes hold a block, so its maximum takes two lane moves.  64 requests'
// 9 kept rows of 36 layers (8 kv heads, d = 128; 107 MB) 28 us, 3.8 TB/s; 12,000 prompt
// rows of 4 layers (249 MB) 56 us, 4.4 TB/s (32 and 62 with integer divisions, exchanges
// through the LDS and 256 threads).  kv_load_mx4_kernel 5.0 TB/s on 191 and 265 MB.
#include <algorithm>
#include <climits>

#include "sg_common.h"

namespace sg {
namespace {

constexpr int kPackThreads = 512;
constexpr int kPackRows = 16;    // kept rows of a workgroup
constexpr int kPackBatch = 4;    // 16-byte chunks a thread loads before it packs any

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
using GlobalU4 = __attribute__((address_space(1))) u32x4;

// |x| of both halves of a word; the larger one as fp32 bits.
__device__ __forceinline__ uint32_t abs_max_bits(uint32_t w) {
  return max((w << 16) & 0x7fffffffu, w & 0x7fff0000u);
}

// (By value: a bit cast of a vector's element takes its first one.)
__device__ __forceinline__ bf16x2 as_pair(uint32_t w) { return __builtin_bit_cast(bf16x2, w); }

// The eight values of v packed against the block scale of the four lanes that
// hold the block; scale byte in `scale`.
__device__ __forceinline__ uint32_t pack8(u32x4 v, uint32_t& scale) {
  uint32_t m = max(max(abs_max_bits(v[0]), abs_max_bits(v[1])),
                   max(abs_max_bits(v[2]), abs_max_bits(v[3])));
  m = max(m, lane_swap<kSwap1>(m));
  m = max(m, lane_swap<kSwap2>(m));
  const bool bad = m >= 0x7f800000u;
  const int e = static_cast<int>((m + 0x1fffffu) >> 23) - 2;
  scale = static_cast<uint32_t>(min(max(e, 1), 252));
  const float s = __uint_as_float(scale << 23);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, as_pair(v[0]), s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, as_pair(v[1]), s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, as_pair(v[2]), s, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, as_pair(v[3]), s, 3);
  if (bad) scale = 255u;
  return bad ? 0u : w;
}

struct PackRequest {
  int keep_len, len, r0, rows;
  int64_t start;
};

__device__ __forceinline__ PackRequest load_request(const SgKvCommitMx4Args& a, int req) {
  PackRequest r;
  r.keep_len = a.keep_len_dev[req];
  r.len = a.lengths_dev[req];
  r.r0 = a.row_offset_dev[req];
  r.rows = a.row_offset_dev[req + 1] - r.r0;
  r.start = a.prefix_start_dev[req];
  return r;
}

// SG_OK when the request's rows may be written, by the same inputs in every
// workgroup (so that all skip it or all write it).  Called by whole workgroups.
__device__ __forceinline__ int check_request(const SgKvCommitMx4Args& a, const PackRequest& r,
                                             const int32_t* keep) {
  if (r.len < 0 || r.keep_len > a.keep_stride || r.keep_len > a.capacity - r.len) return SG_ERANGE;
  bool bad = keep == nullptr && r.keep_len > r.rows;
  if (keep != nullptr) {
    for (int t = threadIdx.x; t < r.keep_len; t += blockDim.x) {
      const int k = keep[t];
      bad = bad || k < 0 || k >= r.rows;
    }
  }
  return __syncthreads_or(bad) ? SG_EINVAL : SG_OK;
}

// Workgroup (x, y, z): kept rows kPackRows * x .. of request y in layer z.
// kUpdate: the grid is one workgroup a request, which also advances its length.
template <bool kUpdate>
__global__ __launch_bounds__(kPackThreads) void kv_commit_mx4_kernel(SgKvCommitMx4Args a) {
  const int req = blockIdx.y;
  const int layer = blockIdx.z;
  const PackRequest r = load_request(a, req);
  const int t0 = blockIdx.x * kPackRows;
  if (t0 >= r.keep_len) return;
  const int32_t* keep =
      a.keep_rows_dev ? a.keep_rows_dev + static_cast<int64_t>(a.keep_stride) * req : nullptr;
  const int code = check_request(a, r, keep);
  if (code != SG_OK) {
    if (threadIdx.x == 0 && blockIdx.x == 0 && layer == 0 && a.status_dev)
      atomicExch(a.status_dev, code);
    return;
  }
  const uint16_t* src[2] = {static_cast<const uint16_t*>(a.k_tree_layers_dev[layer]),
                            static_cast<const uint16_t*>(a.v_tree_layers_dev[layer])};
  unsigned char* codes[2] = {static_cast<unsigned char*>(a.k_code_layers_dev[layer]),
                             static_cast<unsigned char*>(a.v_code_layers_dev[layer])};
  unsigned char* scales[2] = {static_cast<unsigned char*>(a.k_scale_layers_dev[layer]),
                              static_cast<unsigned char*>(a.v_scale_layers_dev[layer])};
  const int per_head = a.head_dim / 8;
  const int per_row = a.num_kv_heads * per_head;
  const int total = min(kPackRows, r.keep_len - t0) * 2 * per_row;  // a multiple of 4
  const int64_t token0 = r.start + r.len + t0;
  // Chunk idx: row t, K or V, head g, piece `chunk` of the head.  Quotients by the
  // reciprocal: idx + 1/2 lies 1/(2 d) from the next multiple's quotient at least, and
  // the host checks that idx < 2^20, for which fp32 errs by less.  (Integer division
  // took as much issue time as the packing: 62 us against 56 for 12,000 rows of 4 layers.)
  const float inv_row = 1.0f / static_cast<float>(2 * per_row);
  const float inv_head = 1.0f / static_cast<float>(per_head);
  struct Place {
    int t, g, chunk;
    bool is_v;
  };
  auto place = [&](int idx) {
    Place p;
    p.t = static_cast<int>((static_cast<float>(idx) + 0.5f) * inv_row);
    const int rem = idx - p.t * (2 * per_row);
    p.is_v = rem >= per_row;
    const int c = p.is_v ? rem - per_row : rem;
    p.g = static_cast<int>((static_cast<float>(c) + 0.5f) * inv_head);
    p.chunk = c - p.g * per_head;
    return p;
  };
  for (int base = threadIdx.x; base < total; base += kPackBatch * kPackThreads) {
    u32x4 v[kPackBatch];
#pragma unroll
    for (int j = 0; j < kPackBatch; ++j) {
      // Past the end: the first chunk again, stored nowhere.
      const int idx = base + j * kPackThreads;
      const Place p = place(idx < total ? idx : base);
      const int k = keep != nullptr ? keep[t0 + p.t] : t0 + p.t;
      v[j] = *(const GlobalU4*)((p.is_v ? src[1] : src[0]) +
                                static_cast<int64_t>(r.r0 + k) * a.tree_row_stride +
                                p.g * a.tree_head_stride + p.chunk * 8);
    }
#pragma unroll
    for (int j = 0; j < kPackBatch; ++j) {
      const int idx = base + j * kPackThreads;
      const Place p = place(idx < total ? idx : base);
      uint32_t scale;
      const uint32_t word = pack8(v[j], scale);
      if (idx >= total) continue;
      *reinterpret_cast<uint32_t*>((p.is_v ? codes[1] : codes[0]) + p.g * a.code_head_stride +
                                   (token0 + p.t) * a.code_token_stride + 4 * p.chunk) = word;
      if ((p.chunk & 3) == 0)
        ((p.is_v ? scales[1] : scales[0]) + p.g * a.scale_head_stride +
         (token0 + p.t) * a.scale_token_stride)[p.chunk >> 2] = static_cast<unsigned char>(scale);
    }
  }
  if constexpr (kUpdate) {
    __syncthreads();
    if (threadIdx.x == 0) a.lengths_dev[req] = r.len + r.keep_len;
  }
}

// Advances the lengths after a launch of several workgroups a request.
__global__ __launch_bounds__(64) void kv_commit_mx4_lengths_kernel(SgKvCommitMx4Args a) {
  const int req = blockIdx.x;
  const PackRequest r = load_request(a, req);
  if (r.keep_len <= 0) return;
  const int32_t* keep =
      a.keep_rows_dev ? a.keep_rows_dev + static_cast<int64_t>(a.keep_stride) * req : nullptr;
  if (check_request(a, r, keep) != SG_OK) return;
  if (threadIdx.x == 0) a.lengths_dev[req] = r.len + r.keep_len;
}

// Eight values (a 4-byte word of codes, 16 bytes out) a lane and step.
__global__ __launch_bounds__(256) void kv_load_mx4_kernel(
    const unsigned char* __restrict__ codes, int64_t code_outer, int64_t code_token,
    const unsigned char* __restrict__ scales, int64_t scale_outer, int64_t scale_token,
    int tokens, int words, uint16_t* __restrict__ out, int64_t out_outer, int64_t out_token,
    int64_t total) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < total;
       i += step) {
    const int64_t row = i / words;
    const int w = static_cast<int>(i - row * words);
    const int64_t o = row / tokens;
    const int64_t t = row - o * tokens;
    const uint32_t c =
        *reinterpret_cast<const uint32_t*>(codes + o * code_outer + t * code_token + 4 * w);
    const uint32_t b = scales[o * scale_outer + t * scale_token + (w >> 2)];
    const float s = __uint_as_float(b << 23);  // 255: infinite, which converts to NaN
    uint4 v;
    v.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0));
    v.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1));
    v.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2));
    v.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3));
    *reinterpret_cast<uint4*>(out + o * out_outer + t * out_token + 8 * w) = v;
  }
}

}  // namespace
}  // namespace sg

extern "C" int sg_kv_commit_mx4(const SgKvCommitMx4Args* args, sg_stream_t stream) {
  using namespace sg;
  clear_error();
  SG_REQUIRE(args != nullptr, "null SgKvCommitMx4Args");
  const SgKvCommitMx4Args& a = *args;
  SG_REQUIRE(a.num_layers >= 0 && a.num_requests >= 0, "negative sizes");
  if (a.num_layers == 0 || a.num_requests == 0) return SG_OK;
  SG_REQUIRE(a.num_kv_heads >= 1 && a.head_dim >= 32 && a.head_dim % 32 == 0,
             "head_dim must be a positive multiple of 32");
  SG_REQUIRE(a.capacity >= 1 && a.keep_stride >= 1, "capacity and keep_stride must be positive");
  SG_REQUIRE(a.tree_row_stride % 8 == 0 && a.tree_head_stride % 8 == 0,
             "tree strides must be multiples of 8 elements (16-byte rows)");
  SG_REQUIRE(a.code_head_stride % 4 == 0 && a.code_token_stride % 4 == 0,
             "code strides must be multiples of 4 bytes");
  SG_REQUIRE(a.k_code_layers_dev && a.k_scale_layers_dev && a.v_code_layers_dev &&
                 a.v_scale_layers_dev && a.k_tree_layers_dev && a.v_tree_layers_dev &&
                 a.row_offset_dev && a.keep_len_dev && a.prefix_start_dev && a.lengths_dev,
             "null device pointer");
  SG_REQUIRE(a.num_requests <= 65535 && a.num_layers <= 65535,
             "at most 65535 requests and layers per call");
  // Chunk indices of one workgroup are divided in fp32.
  SG_REQUIRE(static_cast<int64_t>(kPackRows) * 2 * a.num_kv_heads * (a.head_dim / 8) <
                 (int64_t{1} << 20),
             "num_kv_heads * head_dim must be below 2^18");
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const unsigned blocks = (static_cast<unsigned>(a.keep_stride) + kPackRows - 1) / kPackRows;
  const dim3 grid(blocks, a.num_requests, a.num_layers);
  if (blocks == 1 && a.num_layers == 1) {
    kv_commit_mx4_kernel<true><<<grid, dim3(kPackThreads), 0, s>>>(a);
    SG_LAUNCH_CHECK();
    return SG_OK;
  }
  // The lengths advance in a second launch, after every workgroup has read them.
  kv_commit_mx4_kernel<false><<<grid, dim3(kPackThreads), 0, s>>>(a);
  SG_LAUNCH_CHECK();
  kv_commit_mx4_lengths_kernel<<<dim3(a.num_requests), dim3(64), 0, s>>>(a);
  SG_LAUNCH_CHECK();
  return SG_OK;
}

extern "C" int sg_kv_load_mx4(const void* codes_dev, int64_t code_outer_stride,
                              int64_t code_token_stride, const void* scales_dev,
                              int64_t scale_outer_stride, int64_t scale_token_stride,
                              int32_t outer, int32_t tokens, int32_t head_dim, void* out_dev,
                              int64_t out_outer_stride, int64_t out_token_stride,
                              sg_stream_t stream) {
  using namespace sg;
  clear_error();
  SG_REQUIRE(outer >= 0 && tokens >= 0, "negative sizes");
  SG_REQUIRE(head_dim >= 32 && head_dim % 32 == 0, "head_dim must be a positive multiple of 32");
  if (outer == 0 || tokens == 0) return SG_OK;
  SG_REQUIRE(codes_dev && scales_dev && out_dev, "null device pointer");
  SG_REQUIRE((code_outer_stride | code_token_stride) % 4 == 0 &&
                 (reinterpret_cast<uintptr_t>(codes_dev) & 3) == 0,
             "codes must be 4-byte aligned, their strides multiples of 4 bytes");
  SG_REQUIRE((out_outer_stride | out_token_stride) % 8 == 0 &&
                 (reinterpret_cast<uintptr_t>(out_dev) & 15) == 0,
             "out must be 16-byte aligned, its strides multiples of 8 elements");
  const int words = head_dim / 8;
  const int64_t total = static_cast<int64_t>(outer) * tokens * words;
  const int64_t blocks = std::min<int64_t>((total + 255) / 256, 1 << 16);
  kv_load_mx4_kernel<<<dim3(static_cast<unsigned>(blocks)), dim3(256), 0,
                       static_cast<hipStream_t>(stream)>>>(
      static_cast<const unsigned char*>(codes_dev), code_outer_stride, code_token_stride,
      static_cast<const unsigned char*>(scales_dev), scale_outer_stride, scale_token_stride,
      tokens, words, static_cast<uint16_t*>(out_dev), out_outer_stride, out_token_stride, total);
  SG_LAUNCH_CHECK();
  return SG_OK;
}
