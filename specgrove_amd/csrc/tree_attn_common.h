// Pieces shared by the packed tree attention kernels: the records of a plan,
// the layouts of an unit's LDS tiles and of its partial results, and the
// checks of a unit against the call's metadata.
#pragma once

#include <functional>
#include <vector>

#include "sg_common.h"

namespace sg {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(16))) float floatx16;
typedef __attribute__((ext_vector_type(4))) short short4_t;
typedef __attribute__((ext_vector_type(8))) short short8_t;
typedef __attribute__((address_space(3))) short4_t lds_short4;

constexpr int kQPerUnit = 128;
constexpr int kTileKeys = 32;                   // keys per tile: one 32-key MFMA block
constexpr int kMaxTreeRows = 256;
constexpr int kAncWords = kMaxTreeRows / 32;
constexpr int kMergeThreads = 256;
constexpr int32_t kPlanMagic = 0x53475041;  // "SGPA"
constexpr int kMaxGroup = 16;               // query heads per kv head
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazyLog2 = 8.0f;  // softmax reference point moves after a 2^8 growth

constexpr int kListsPerCU = 2;                  // resident workgroups per CU
constexpr int kDefaultCUs = 256;

struct PlanHeader {
  int32_t magic;
  int32_t num_units;
  int32_t num_merges;
  int32_t rows_per_tile;
  int32_t head_dim;
  int32_t group;
  int32_t num_partials;
  int32_t num_bins;       // work lists = workgroups of the attention kernel
  int32_t num_requests;   // n and R = row_offset[n] of the wave the plan was built for
  int32_t num_rows;
  int32_t num_kv_heads;
  int32_t unit_rows;      // most rows of a unit; 0: not known (plans made before the field)
  uint64_t meta_hash;     // FNV-1a over row_offset[0..n] and prefix_len[0..n-1]
  int32_t reserved[2];
};
static_assert(sizeof(PlanHeader) == 64, "plan header is 64 bytes");

struct AttnUnit {
  int32_t req;
  int32_t kv_head;
  int32_t row_begin;
  int32_t row_count;
  int32_t key_begin;
  int32_t key_end;
  int32_t partial;        // partial slot of this unit, -1 when unsplit
  int32_t flags;          // bit 0: attend to the request's tree rows; bit 1: rows
                          // split, K/V shared with sibling units (no nt hint)
  int32_t group;          // split group (merge record index), -1 when unsplit
  int32_t num_splits;     // units in the group
  int32_t first_partial;  // partial slot of the group's first unit
  int32_t pad;
};
static_assert(sizeof(AttnUnit) == 48, "unit record is 48 bytes");

struct MergeGroup {
  int32_t req;
  int32_t kv_head;
  int32_t row_begin;
  int32_t row_count;
  int32_t first_partial;
  int32_t num_partials;
  int32_t pad0;
  int32_t pad1;
};

__host__ __device__ constexpr size_t partial_floats(int head_dim) {
  return static_cast<size_t>(kQPerUnit) * (head_dim + 2);
}

__host__ __device__ constexpr int merge_blocks_per_group(int head_dim) {
  return (head_dim / 4) * kQPerUnit / kMergeThreads;
}

// LDS row of key k inside its 32-key block (inverse of pi).
__device__ __forceinline__ int key_slot(int k) {
  return 8 * ((k >> 2) & 3) + 4 * (k >> 4) + (k & 3);
}

// Key held by LDS row i of a 32-key K block (pi).
__device__ __forceinline__ int key_pi(int i) {
  return 16 * ((i >> 2) & 1) + 4 * (i >> 3) + (i & 3);
}

// XOR swizzles of the 16-byte chunks of LDS row r, chosen by exhaustive check
// of every read pattern of this kernel against both 32- and 64-bank LDS:
//   K rows (ds_read_b128, 16 consecutive rows at one chunk): r & 15 (D=128),
//     r & 7 (D=64, 8 chunks per row);
//   V rows (ds_read_b64_tr_b16, 4 consecutive rows at 2-4 adjacent chunks):
//     4*(r&3) + 2*((r>>1)&1) (D=128), 2*(r&3) (D=64).
template <int D>
__host__ __device__ constexpr int swz_k(int r) {
  return D == 128 ? (r & 15) : (r & 7);
}
template <int D>
__host__ __device__ constexpr int swz_v(int r) {
  return D == 128 ? 4 * (r & 3) + 2 * ((r >> 1) & 1) : 2 * (r & 3);
}

__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) char*)p));
}

// max / sum of a value with the same lane of the other 32-lane half.
__device__ __forceinline__ float half_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v),
                                                  false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v),
                                                  false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ bf16x8 as_bf16x8(uint4 v) { return __builtin_bit_cast(bf16x8, v); }

__device__ __forceinline__ uint4 zero4() { return make_uint4(0u, 0u, 0u, 0u); }

// Per-wave attention state: one query column per lane pair.
template <int D>
struct WaveState {
  float m;  // running max of raw scores
  float l;  // running sum of exp2((s - m) * c2)
  floatx16 acc[D / 32];
};

// The unit's request, kv head and partial slot exist in this call (checked
// before any of them indexes memory).
template <int D>
__device__ __forceinline__ bool unit_indices_valid(const SgTreeAttnArgs& a, const AttnUnit& u) {
  return u.req >= 0 && u.req < a.num_requests && u.kv_head >= 0 &&
         u.kv_head < a.num_kv_heads &&
         (u.partial < 0 ||
          static_cast<size_t>(u.partial) < a.workspace_bytes / (sizeof(float) * partial_floats(D)));
}

// The unit's rows and key range lie inside request req's rows and cached
// prefix as the metadata of this call gives them, and the unit that covers
// the tree rows ends the key range exactly at the prefix length.
__device__ __forceinline__ bool unit_matches(const SgTreeAttnArgs& a, const AttnUnit& u, int r0,
                                             int n, int prefix_len) {
  return r0 >= 0 && n >= 1 && n <= kMaxTreeRows && r0 <= a.num_rows - n && u.row_begin >= 0 &&
         u.row_count >= 1 && u.row_begin + u.row_count <= n && u.key_begin >= 0 &&
         u.key_begin <= u.key_end && u.key_end <= prefix_len &&
         ((u.flags & 1) == 0 || u.key_end == prefix_len);
}

// Marks a mismatched unit: the status word, and NaN in its output rows (or in
// its split partial, which the merge then turns into NaN output).
template <int D>
__device__ void poison_unit(const SgTreeAttnArgs& a, const AttnUnit& u, int r0) {
  const int tid = threadIdx.x;
  if (tid == 0 && a.status_dev != nullptr) *a.status_dev = SG_EINVAL;
  const float qnan = __builtin_nanf("");
  if (u.partial >= 0) {
    float* part = static_cast<float*>(a.workspace_dev) + partial_floats(D) * u.partial;
    for (int k = tid; k < static_cast<int>(partial_floats(D)); k += blockDim.x)
      part[k] = (k >= kQPerUnit * D && k < kQPerUnit * (D + 1)) ? 0.0f : qnan;
    return;
  }
  const int G = a.num_q_heads / a.num_kv_heads;
  uint16_t* out = static_cast<uint16_t*>(a.out_dev);
  for (int k = tid; k < u.row_count * G * D; k += blockDim.x) {
    const int rr = k / (G * D);
    const int h = (k / D) % G;
    const int64_t row = static_cast<int64_t>(r0) + u.row_begin + rr;
    if (r0 < 0 || row < 0 || row >= a.num_rows) continue;
    out[row * a.out_row_stride + static_cast<int64_t>(u.kv_head * G + h) * a.out_head_stride +
        k % D] = 0x7fc0;  // bf16 quiet NaN
  }
}

// One node per thread (n <= kMaxTreeRows <= threads): its parent.
__device__ __forceinline__ int load_parent(const SgTreeAttnArgs& a, int r0, int n) {
  const int tid = threadIdx.x;
  return tid < n ? a.parent_dev[r0 + tid] : -1;
}

// Ancestor-or-self bitsets of the tile's rows (request-local numbering), from every
// thread's load_parent().  A
// row's walk to its root takes a run of consecutive nodes (parent = node - 1)
// at a step: every step is a dependent LDS read and eight words of bits, and
// a 256-row prompt chunk walked node by node spent ~17 us here, an eighth of
// its unit.  Runs are found inside groups of 64 nodes (a ballot per wave), so
// a chain of 256 takes four steps and a bushy tree never more than its depth.
// With the tree tiles that a row tile cannot see left out, eight 256-row
// chunks at 483-3,006 cached tokens (32 q / 8 kv heads): 138 -> 110 us.
// For workgroups of at least kMaxTreeRows threads; s_run [kMaxTreeRows] is
// scratch (first node of each node's run, and that node's parent), s_anc
// [kQPerUnit] is read after the caller's next barrier.
__device__ __forceinline__ void build_ancestors(const AttnUnit& u, int p, int2* s_run,
                                                uint32_t (*s_anc)[kAncWords]) {
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  if (tid < kMaxTreeRows) {
    const uint64_t linked = __ballot(lane > 0 && p == tid - 1);
    // The run starts at the highest unlinked lane at or below this one.
    const int start = 63 - __builtin_clzll(~linked & (~0ull >> (63 - lane)));
    const int above = __shfl(p, start);
    s_run[tid] = make_int2((tid & ~63) + start, above);
  }
  for (int k = tid; k < kQPerUnit * kAncWords; k += blockDim.x) (&s_anc[0][0])[k] = 0u;
  __syncthreads();
  if (tid < u.row_count) {
    int node = u.row_begin + tid;
    uint32_t bits[kAncWords];
#pragma unroll
    for (int w = 0; w < kAncWords; ++w) bits[w] = 0u;
    for (int guard = 0; node >= 0 && guard < kMaxTreeRows; ++guard) {
      const int2 run = s_run[node];
#pragma unroll
      for (int w = 0; w < kAncWords; ++w) {
        // Bits run.x .. node of word w.
        const int lo = max(run.x - 32 * w, 0), hi = min(node - 32 * w, 31);
        bits[w] |= lo <= hi ? (0xffffffffu << (lo & 31)) & (0xffffffffu >> ((31 - hi) & 31)) : 0u;
      }
      node = (run.y < run.x) ? run.y : -1;
    }
#pragma unroll
    for (int w = 0; w < kAncWords; ++w) s_anc[tid][w] = bits[w];
  }
}

// Host checks that every form of the attention shares (head counts, sizes, the
// plan's header, device pointers, the strides of q, the tree rows and out), and
// what the kernels get from the plan's host copy.
struct AttnCall {
  const MergeGroup* merge_groups;  // on the device, nullptr when not known
  const AttnUnit* direct;          // unit records when every list is one unit
  int unit_rows;                   // most rows of a unit, 0 when not known
};
int check_attn_call(const SgTreeAttnArgs& a, AttnCall* call);

// A wave to be planned: into how many prefix pieces each request's units are cut, which
// requests' large units are cut by rows, and what a unit costs (in any measure, from its
// rows and 32-key tiles).  lists: 0, or the number of work lists to pack the units onto.
// pieces_apart: pieces of one prefix need not share an XCD (they share no keys).
struct PlanWave {
  int32_t num_requests;
  const int32_t* row_offset;
  const int32_t* prefix_len;
  int32_t num_q_heads, num_kv_heads, head_dim;
  int64_t lists = 0;
  std::vector<int> splits;
  std::vector<char> split_rows;
  std::function<int64_t(int, int64_t)> unit_cost;
  bool pieces_apart = false;
};
struct PlanOut {
  void* host;  // nullptr: a size query
  size_t capacity;
  size_t* bytes;
  int32_t* units;
  int32_t* merges;
  size_t* workspace_bytes;
};
int check_plan_wave(const PlanWave& wave, const PlanOut& out);
// The plan's records (units, merge groups, work lists) into out.
int emit_plan(const PlanWave& wave, const PlanOut& out);

// Combines the plan's split partials (after the attention kernel).
int launch_attn_merge(const SgTreeAttnArgs& a, const MergeGroup* groups, hipStream_t stream);

}  // namespace sg
