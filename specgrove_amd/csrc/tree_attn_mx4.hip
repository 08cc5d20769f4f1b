// Packed tree attention over a prefix held in 4 bits (e2m1 codes with a
// power-of-two scale for 32 values of a row; mx4_cache.hip).
//
// Row k of request i attends to request i's cached prefix and to its own tree
// rows that are ancestors of k or k itself, with softmax(q.k * scale) weights;
// plans, units, split partials and their merge are those of tree_attn.hip.  The
// prefix's values are bf16 values, so the products are the bf16 kernel's over
// the unpacked cache.
//
// K is multiplied as it is held: v_mfma_scale_f32_32x32x64_f8f6f4 takes e2m1
// elements with a power-of-two scale for 32 of them, so S^T = K Q^T needs no
// unpacking and no LDS, if Q is in 8 bits.  A bf16 value q is held as two e4m3 values
// with scales for 32 columns: hi is q rounded to 4 significant bits, lo = q - hi has 4
// at most and a scale 2^5 smaller; two products each, in the time of the bf16 ones.
// q = hi + lo exactly from 2^-14 of its block's largest value on; below that hi is one
// of e4m3's subnormals or 0 and lo is rounded to multiples of 2^-21 of a power of two
// that the largest reaches, so the error is at most 2^-22 of the largest.
//
// V is unpacked to bf16 (gfx950: two values an instruction, scale included) into
// LDS and read transposed (ds_read_b64_tr_b16) for O^T += V^T P^T with
// v_mfma_f32_32x32x16_bf16, as in tree_attn.hip.
//
// What is narrower than fp32 in between.  The instruction adds the products of 8
// columns at a time, cut towards 0 to multiples of 2^(e - 13), e the largest sum of a
// column's two exponents (measured; the 8-sums and the accumulator are added in fp32).
// 7 products of 8 can lose, so a score is off by less than 2^-10 of sum |k q| where one
// of every 8 products is some hundred times the others, by 2^-16 of it at most and
// 2^-20 in the mean over Gaussian rows.  Kept, since K's own 4 bits move
// a value by up to a fifth: products in bf16 (6 to 22 % more time, under "Tried") would
// not bring the result nearer to the rows that were packed.  Probabilities are
// rounded to bf16 for the matrix product, as in tree_attn.hip (their sum is not): each
// by 2^-8 of it at most, and the output's error against 64 bits is 1.4 times that of
// its own rounding; V in fp16 would lose its scales' range, P in two terms would take
// the larger of the two products twice.
//
// Waves.  A wave takes one q-group of 32 query vectors over 32-key tiles; 1 q-group:
// four key streams, each wave with V tiles of its own and no barrier; 2: two
// streams; 3-4: one.  There the workgroup unpacks 64 keys of V at a time together,
// a piece a thread, into one of two stages (one barrier for 64 keys).  Codes are
// loaded two tiles (stages) ahead into registers: a tile is 4.3 KB.  K goes from there
// into the products, for 3-4 q-groups through LDS, where all waves take it.  Two
// workgroups share a CU; streams are merged at the end.
//
// Measured (64 requests of 16,384 cached tokens, 32 q / 8 kv heads, d = 128; 1 / 16 /
// 32 rows each): 240 / 363 / 597 us, that is 4.8 / 3.1 / 1.9 TB/s of codes and scales
// and 72 / 757 / 921 TFLOP/s.  One row a request is bound by the cache's bytes, 32
// by issue: a wave and tile take 119 vector instructions and 12 products, of which a
// wave alone on its SIMD can overlap little (450 us for half the requests, one workgroup
// a CU).  Tried, at 234 / 365 / 619 us: K and V unpacked to bf16 by the workgroup, 406 /
// 444 / 702; by each wave for itself, 249 / 470 / 873; the products of a tile issued
// before the softmax of the one before it, 583 / 381 / 672 (spills at one row); all of V
// read before the softmax, 314 / 369 / 620; K two tiles ahead for 3-4 q-groups too
// (spills), 243 / 433 / 664; s_setprio around the products, no difference.
#include <algorithm>
#include <cmath>
#include <map>
#include <type_traits>
#include <vector>

#include "tree_attn_common.h"

namespace sg {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(2))) short short2_t;
typedef __attribute__((ext_vector_type(8))) int intx8;

__device__ __forceinline__ bf16x2 as_pair(uint32_t w) { return __builtin_bit_cast(bf16x2, w); }

// XOR swizzle of the 16-byte chunks of V's LDS row r.  The transposed reads take 64
// bytes of each of four consecutive rows: bits 2 and 3 (bit 2 at D = 64, where two
// rows fill the banks) put those on different banks.  The unpacked writes take one
// chunk of each block of four (two) consecutive rows: the low bits.  (4 (r & 3) +
// 2 (r >> 1 & 1), right for the reads alone, spent half of the LDS's active cycles
// on conflicts of the writes.)  Both repeat every four rows.
template <int D>
__host__ __device__ constexpr int swz_kc(int r) {  // of K's codes: 16 rows at one chunk
  return D == 128 ? (r >> 2) & 3 : (r >> 3) & 1;
}
template <int D>
__host__ __device__ constexpr int swz_w(int r) {
  return D == 128 ? 5 * (r & 3) : 5 * ((r >> 1) & 1);
}

// 16-byte chunk c (8 values) of 32 unpacked ones, from code word `w` of a block.
__device__ __forceinline__ uint4 unpack8(uint32_t w, float scale) {
  uint4 v;
  v.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
  v.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
  v.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
  v.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
  return v;
}

// Bit mask of a word's halves that are infinities or NaNs, as a word of which
// those halves are all ones.
__device__ __forceinline__ uint32_t nonfinite_halves(uint32_t w) {
  const uint32_t lo = (w & 0x7f80u) == 0x7f80u ? 0xffffu : 0u;
  const uint32_t hi = (w & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u;
  return lo | hi;
}

// The call's arguments where the launch put them.  What is read through a fresh()
// pointer is loaded there and then: kept in registers from the kernel's start,
// the arguments filled the scalar ones, and every load of the loop moved 30 of
// their words back from vector lanes first.
using ArgsIn = const __attribute__((address_space(4))) SgTreeAttnMx4Args*;
__device__ __forceinline__ ArgsIn fresh(ArgsIn p) {
  asm volatile("" : "+s"(p));
  return p;
}
// A scalar address that is not put together again from its parts at every use.
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
using GlobalBytes = const __attribute__((address_space(1))) unsigned char*;
using GlobalU4 = const __attribute__((address_space(1))) u32x4*;
__device__ __forceinline__ GlobalBytes settled(const unsigned char* p) {
  GlobalBytes g = (GlobalBytes)p;
  asm volatile("" : "+s"(g));
  return g;
}

// LDS of a workgroup: 8 KB of V (D = 128) a wave, after the last tile the merge
// scratch and the output staging; and the tree's tables.
template <int D>
struct Shared {
  static constexpr int kSlot = (2 + D / 2) * 64 * 4;   // a wave's state
  static constexpr int kStage = 32 * (2 * D + 16);     // a wave's output rows
  static constexpr int kBytes = kWaves * kSlot;
  static_assert(kBytes >= kWaves * kTileKeys * 2 * D && kBytes >= kSlot * 2 + kStage * 2 &&
                    kBytes >= kStage * 4,
                "every use of the buffer must fit");
  __align__(1024) unsigned char buf[kBytes];
  uint32_t anc[kQPerUnit][kAncWords];
  int2 run[kMaxTreeRows];
};

// One unit.  kShared: of 2-4 q-groups, V unpacked by the workgroup; kBoth: of 3-4, a
// wave takes both tiles of a stage.
template <int D, bool kShared, bool kBoth>
__device__ __forceinline__ void attn_unit_mx4(const SgTreeAttnMx4Args& args, ArgsIn in,
                                              const AttnUnit& u, Shared<D>& sh) {
  const SgTreeAttnArgs& a = args.attn;
  constexpr int DB = D / 32;                  // PV blocks of 32 columns
  constexpr int ROWB = D * 2;                 // bytes of an LDS row
  constexpr int P = D / 64;                   // 16-byte pieces of codes a lane loads of K (and V)
  constexpr int kPitch = ROWB + 16;

  // Query heads of a kv head: 1, 2, 4, 8 or 16.
  const int g_bits = __builtin_ctz(static_cast<unsigned>(a.num_q_heads / a.num_kv_heads));
  const int G = 1 << g_bits;
  // Opaque, so that what follows from it is not kept in registers from one unit
  // of a list to the next.
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5;
  const int col = lane & 31;
  if (!unit_indices_valid<D>(a, u)) {
    if (tid == 0 && a.status_dev != nullptr) *a.status_dev = SG_EINVAL;
    return;
  }
  const int r0 = a.row_offset_dev[u.req];
  const int n = a.row_offset_dev[u.req + 1] - r0;
  if (!unit_matches(a, u, r0, n, a.prefix_len_dev[u.req])) {
    poison_unit<D>(a, u, r0);
    return;
  }
  const int nq = (u.row_count * G + 31) / 32;   // q-groups in use, 1..4
  constexpr int streams = kBoth ? 1 : kShared ? 2 : 4;  // key streams of each
  const int qg = wave % nq;
  const int ks = wave / nq;
  const bool active = ks < streams;
  const int m = qg * 32 + col;                // query vector inside the unit
  const int r_local = m >> g_bits;
  const int head = u.kv_head * G + (m - r_local * G);
  const bool q_valid = active && r_local < u.row_count;
  const int64_t row = static_cast<int64_t>(r0) + u.row_begin + r_local;
  const int g = u.kv_head;
  const bool do_tree = (u.flags & 1) != 0;

  // The parents are on their way before the prefix's first codes: loads return in
  // order.  (Q and the tree's first tile loaded here too spilled, and cost 3 us.)
  const int tree_keys = do_tree ? u.row_begin + u.row_count : 0;
  const int parent = do_tree ? load_parent(a, r0, n) : -1;
  // Q, bf16: piece [j][b][e] is columns 64 j + 32 b + 16 half + 8 e .. +7.
  const uint16_t* const q_row = static_cast<const uint16_t*>(a.q_dev) + row * a.q_row_stride +
                                static_cast<int64_t>(head) * a.q_head_stride;
  auto q_piece = [&](int j, int b, int e) {
    return q_valid ? *reinterpret_cast<const uint4*>(q_row + 64 * j + 32 * b + 16 * half + 8 * e)
                   : zero4();
  };
  // Tree tile t: K of key pi(col) in the columns of q_raw, and V as it is written to LDS.
  constexpr int kBlocks = D / 32;             // 32-column blocks of a row
  const int v_row = lane / kBlocks;           // of piece 0; piece i: + 64 / kBlocks
  const int v_blk = lane % kBlocks;
  constexpr int kVStep = 64 / kBlocks;
  const int k_key = key_pi(col);
  struct TreeTile {
    uint4 k[P][2][2], v[P][4];
  };
  auto load_tree = [&](int t, TreeTile& tile) {
    const int64_t tree0 = g * a.tree_head_stride + static_cast<int64_t>(r0) * a.tree_row_stride;
    const int key0 = kTileKeys * t;
    const uint16_t* kr = static_cast<const uint16_t*>(a.k_tree_dev) + tree0 +
                         static_cast<int64_t>(min(key0 + k_key, n - 1)) * a.tree_row_stride +
                         16 * half;
#pragma unroll
    for (int j = 0; j < P; ++j)
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          tile.k[j][b][e] = *reinterpret_cast<const uint4*>(kr + 64 * j + 32 * b + 8 * e);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const uint16_t* vr =
          static_cast<const uint16_t*>(a.v_tree_dev) + tree0 +
          static_cast<int64_t>(min(key0 + v_row + kVStep * i, n - 1)) * a.tree_row_stride +
          32 * v_blk;
#pragma unroll
      for (int c = 0; c < 4; ++c) tile.v[i][c] = *reinterpret_cast<const uint4*>(vr + 8 * c);
    }
  };
  // Codes and scales of this lane.  K: of key pi(col) of a tile, piece j holds
  // columns 64 j + 32 half .. +31, an operand of product j.  V: piece i is 32
  // columns of a row, of a tile or (shared) of a window's 64 keys.
  const int prefix_keys = u.key_end - u.key_begin;
  const int tiles = active ? (prefix_keys + kTileKeys - 1) / kTileKeys : 0;
  const int64_t prefix0 = a.prefix_start_dev[u.req] + u.key_begin;
  const int64_t code0 = g * a.cache_head_stride + prefix0 * a.cache_token_stride;
  const int64_t scale0 = g * args.scale_head_stride + prefix0 * args.scale_token_stride;
  const GlobalBytes k_codes =
      settled(static_cast<const unsigned char*>(a.k_cache_dev) + code0);
  const GlobalBytes v_codes =
      settled(static_cast<const unsigned char*>(a.v_cache_dev) + code0);
  const GlobalBytes k_scales =
      settled(static_cast<const unsigned char*>(args.k_scale_dev) + scale0);
  const GlobalBytes v_scales =
      settled(static_cast<const unsigned char*>(args.v_scale_dev) + scale0);
  uint32_t c_stride = static_cast<uint32_t>(a.cache_token_stride);
  uint32_t s_stride = static_cast<uint32_t>(args.scale_token_stride);
  asm volatile("" : "+s"(c_stride), "+s"(s_stride));
  constexpr int kWindow = 2 * kTileKeys;      // keys of a shared stage
  const int w_row = tid / kBlocks;            // of a window's piece, below kWindow
  const bool w_piece = kWindow * kBlocks >= kThreads || wave < kWindow * kBlocks / 64;
  struct Raw {
    u32x4 c[P];
    uint32_t s[P];
  };
  // Offsets inside a whole tile (window).
  const uint32_t kc_at = k_key * c_stride + 16 * half, ks_at = k_key * s_stride + half;
  uint32_t vc_at[P], vs_at[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    vc_at[i] = (kShared ? w_row : v_row + kVStep * i) * c_stride + 16 * v_blk;
    vs_at[i] = (kShared ? w_row : v_row + kVStep * i) * s_stride + v_blk;
  }
  // Keys past the range read the last valid one: its score is masked, its
  // probability 0.
  auto load_k = [&](int t, Raw& r) {
    const GlobalBytes c = k_codes + static_cast<int64_t>(t) * kTileKeys * c_stride;
    const GlobalBytes s = k_scales + static_cast<int64_t>(t) * kTileKeys * s_stride;
    uint32_t ca = kc_at, sa = ks_at;
    const int last = prefix_keys - 1 - t * kTileKeys;
    if (last < kTileKeys - 1) {
      const uint32_t key = min(k_key, last);
      ca = key * c_stride + 16 * half;
      sa = key * s_stride + half;
    }
#pragma unroll
    for (int j = 0; j < P; ++j) {
      r.c[j] = *(GlobalU4)(c + ca + 32 * j);
      r.s[j] = s[sa + 2 * j];
    }
  };
  // Tile t's V (private), window t's piece of this thread (shared).
  auto load_rows = [&](GlobalBytes codes, GlobalBytes scales, int t, Raw& r) {
    constexpr int kKeys = kShared ? kWindow : kTileKeys;
    if (kShared && !w_piece) return;
    const GlobalBytes c = codes + static_cast<int64_t>(t) * kKeys * c_stride;
    const GlobalBytes s = scales + static_cast<int64_t>(t) * kKeys * s_stride;
    const int last = prefix_keys - 1 - t * kKeys;
#pragma unroll
    for (int i = 0; i < (kShared ? 1 : P); ++i) {
      uint32_t ca = vc_at[i], sa = vs_at[i];
      if (last < kKeys - 1) {
        const uint32_t key = min(kShared ? w_row : v_row + kVStep * i, last);
        ca = key * c_stride + 16 * v_blk;
        sa = key * s_stride + v_blk;
      }
      r.c[i] = *(GlobalU4)(c + ca);
      r.s[i] = s[sa];
    }
  };
  auto load_v = [&](int t, Raw& r) { load_rows(v_codes, v_scales, t, r); };
  auto load_kw = [&](int w, Raw& r) { load_rows(k_codes, k_scales, w, r); };  // a window's K
  // rk[p], rv[p]: this wave's tiles (windows) of even (odd) number.
  const int windows = (prefix_keys + kWindow - 1) / kWindow;
  Raw rk[2], rv[2];
  if constexpr (kBoth) {
    if (windows > 0) load_kw(0, rk[0]);
    if (windows > 1) load_kw(1, rk[1]);
  } else {
    if (ks < tiles) load_k(ks, rk[0]);
    if (ks + streams < tiles) load_k(ks + streams, rk[1]);
  }
  if constexpr (kShared) {
    if (windows > 0) load_v(0, rv[0]);
    if (windows > 1) load_v(1, rv[1]);
  } else {
    if (ks < tiles) load_v(ks, rv[0]);
    if (ks + streams < tiles) load_v(ks + streams, rv[1]);
  }

  if (do_tree) build_ancestors(u, parent, sh.run, sh.anc);

  // LDS of this wave's V tile.  Chunk c of row r is at c ^ swz(r): a block's chunk c
  // is at its first one's address ^ 16 c.
  unsigned char* const s_v = sh.buf + wave * kTileKeys * ROWB;
  uint32_t v_at[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int r = v_row + kVStep * i;
    v_at[i] = r * ROWB + 16 * ((4 * v_blk) ^ swz_w<D>(r));
  }
  const int gq = lane >> 4;
  const int jj = lane & 15;
  const int rr = jj >> 2;
  const int cc = jj & 3;
  // Of the transposed reads: column block db is at v_read ^ 64 db, and the rows 4 on
  // have the same swizzle.
  const int v_first = 16 * half + rr;
  const int v_read = v_first * ROWB +
                     16 * ((2 * (gq & 1) + (cc >> 1)) ^ swz_w<D>(v_first)) + 8 * (cc & 1);

  const float c2 = a.scale * kLog2e;
  WaveState<D> st;
  st.m = -__builtin_inff();
  st.l = 0.0f;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) st.acc[db][r] = 0.0f;

  auto put_v = [&](const Raw& r) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const float scale = __uint_as_float(r.s[i] << 23);
      const uint32_t w[4] = {r.c[i][0], r.c[i][1], r.c[i][2], r.c[i][3]};
#pragma unroll
      for (int c = 0; c < 4; ++c)
        *reinterpret_cast<uint4*>(s_v + (v_at[i] ^ (16 * c))) = unpack8(w[c], scale);
    }
  };
  // This thread's piece of a window into stage p of two.
  const uint32_t w_at = w_row * ROWB + 16 * ((4 * v_blk) ^ swz_w<D>(w_row));
  auto put_w = [&](const Raw& r, int p) {
    if (!w_piece) return;
    const float scale = __uint_as_float(r.s[0] << 23);  // 255: converts to NaN
    const uint32_t w[4] = {r.c[0][0], r.c[0][1], r.c[0][2], r.c[0][3]};
#pragma unroll
    for (int c = 0; c < 4; ++c)
      *reinterpret_cast<uint4*>(sh.buf + p * kWindow * ROWB + (w_at ^ (16 * c))) =
          unpack8(w[c], scale);
  };
  // Where every wave takes every tile (kBoth), the workgroup brings K into LDS too, as it
  // is held, each thread a piece: waves that loaded whole tiles for themselves had
  // registers for one tile ahead only (16,384 tokens, 32 rows: 631 us, 619 so; with two
  // q-groups it lost, 368 and 410).  K of a window lies behind V's stages: rows of D / 2 bytes whose 16-byte chunk c
  // is at c ^ swz_kc(row), then the scales.
  constexpr int kRowK = D / 2;
  constexpr int kStageK = kWindow * (kRowK + kBlocks);
  unsigned char* const s_k = sh.buf + 2 * kWindow * ROWB;
  static_assert(2 * kWindow * ROWB + 2 * kStageK <= Shared<D>::kBytes, "K's stages must fit");
  auto put_k = [&](const Raw& r, int p) {
    if (!w_piece) return;
    unsigned char* st = s_k + p * kStageK;
    *reinterpret_cast<u32x4*>(st + w_row * kRowK + 16 * (v_blk ^ swz_kc<D>(w_row))) = r.c[0];
    st[kWindow * kRowK + w_row * kBlocks + v_blk] = static_cast<unsigned char>(r.s[0]);
  };
  // This lane's operands of tile i of stage p.
  auto take_k = [&](int p, int i) {
    const unsigned char* st = s_k + p * kStageK;
    const int row = kTileKeys * i + k_key;
    Raw r;
#pragma unroll
    for (int j = 0; j < P; ++j)
      r.c[j] = *reinterpret_cast<const u32x4*>(st + row * kRowK +
                                               16 * ((2 * j + half) ^ swz_kc<D>(row)));
    const unsigned char* sc = st + kWindow * kRowK + row * kBlocks;
    const uint32_t all = D == 128 ? *reinterpret_cast<const uint32_t*>(sc)
                                  : *reinterpret_cast<const uint16_t*>(sc);
#pragma unroll
    for (int j = 0; j < P; ++j) r.s[j] = (all >> (8 * half + 16 * j)) & 0xffu;
    return r;
  };
  // Online softmax of the tile's scores x (masked already): probabilities in x.
  // The reference point st.m moves only when a lane's maximum grew by more than
  // kLazyLog2 in exp2 units (at most 2^kLazyLog2 is exact in bf16 and fp32).
  auto softmax = [&](floatx16& x) {
    float tmax = x[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) tmax = fmaxf(tmax, x[r]);
    tmax = half_max(tmax);
    const float m_new = fmaxf(st.m, tmax);
    if (__ballot((m_new - st.m) * c2 > kLazyLog2)) {
      const float alpha = (st.m == -__builtin_inff())
                              ? 0.0f
                              : __builtin_amdgcn_exp2f((st.m - m_new) * c2);
      st.l *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) st.acc[db][r] *= alpha;
      st.m = m_new;
    }
    const float mc = (st.m == -__builtin_inff()) ? 0.0f : st.m * c2;
    float psum = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      x[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[r], c2, -mc));
      psum += x[r];
    }
    st.l += half_sum(psum);
  };
  // V^T of half c of the tile's keys (a product's 16), at v0.  A wave's LDS accesses
  // run in order, so the reads see the rows that its other lanes wrote before them.
  struct Values {
    short8_t v[DB];
  };
  auto read_v = [&](const unsigned char* v0, int c) {
    Values r;
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      const unsigned char* at = v0 + 8 * c * ROWB + (v_read ^ (64 * db));
      const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)at);
      const short4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(at + 4 * ROWB));
      r.v[db] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    // Keeps the reads here; in the private form that cost registers (268 against
    // 238 us at one row).
    if constexpr (kShared && !kBoth) __builtin_amdgcn_sched_barrier(0);
    return r;
  };
  // O^T += V^T P^T over half c.
  auto pv = [&](const floatx16& x, const Values& r, int c) {
    bf16x8 pf;
#pragma unroll
    for (int e = 0; e < 8; ++e) pf[e] = static_cast<__bf16>(x[8 * c + e]);
#pragma unroll
    for (int db = 0; db < DB; ++db)
      st.acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, r.v[db]), pf,
                                                           st.acc[db], 0, 0, 0);
  };
  // Softmax of the tile's scores x and the product with its V.  The first half of V
  // is read before the softmax, the second while the first is multiplied (read
  // after it, every product waited for its reads).
  auto weigh = [&](floatx16& x, const unsigned char* v0) {
    __builtin_amdgcn_wave_barrier();
    const Values first = read_v(v0, 0);
    softmax(x);
    const Values second = read_v(v0, 1);
    pv(x, first, 0);
    pv(x, second, 1);
    __builtin_amdgcn_wave_barrier();
  };
  // The tile's keys from `limit` on, and those whose bit is off (bit r: this lane's
  // key r), get the score -inf.
  auto mask = [&](floatx16& x, int limit, uint32_t bits) {
    const int mine = limit - 16 * half;  // keys of this lane's 16
    bits &= mine >= 16 ? 0xffffu : mine > 0 ? (1u << mine) - 1u : 0u;
    asm volatile("" : "+v"(bits));
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = ((bits >> r) & 1u) ? x[r] : -__builtin_inff();
  };

  // The request's own rows.  Parents precede their children: no row of the unit
  // sees a tree key behind its last row.
  uint32_t odd_tiles = 0u;  // tree tiles of this wave with a V that is no number
  if (do_tree) {
    __syncthreads();  // the ancestor table is built
    uint4 q_raw[P][2][2];
#pragma unroll
    for (int j = 0; j < P; ++j)
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 2; ++e) q_raw[j][b][e] = q_piece(j, b, e);
    for (int t = active ? ks : kAncWords; kTileKeys * t < tree_keys; t += streams) {
      TreeTile tree;
      load_tree(t, tree);
      const int key0 = kTileKeys * t;
      floatx16 s;
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = 0.0f;
#pragma unroll
      for (int j = 0; j < P; ++j)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                as_bf16x8(tree.k[j][b][e]), as_bf16x8(q_raw[j][b][e]), s, 0, 0, 0);
      uint32_t any = 0u;
#pragma unroll
      for (int i = 0; i < P; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          // A value that is no number would reach every row of the tile through a
          // product with 0: it is added by itself at the end.
          uint32_t w[4] = {tree.v[i][c].x, tree.v[i][c].y, tree.v[i][c].z, tree.v[i][c].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t odd = nonfinite_halves(w[e]);
            any |= odd;
            w[e] &= ~odd;
          }
          *reinterpret_cast<uint4*>(s_v + (v_at[i] ^ (16 * c))) =
              make_uint4(w[0], w[1], w[2], w[3]);
        }
      if (__ballot(any != 0u) != 0) odd_tiles |= 1u << t;
      mask(s, n - key0, sh.anc[r_local][t] >> (16 * half));
      weigh(s, s_v);
    }
    if (kShared) __syncthreads();  // the stages are free
  }

  // The query vector in two 8-bit terms.  Product j takes columns 64 j .. +63: this
  // lane's bytes 0-15 are columns 64 j + 16 half .. +15, bytes 16-31 those 32 on;
  // the scale of block b (32 columns) is read from lane half b.
  intx8 q_hi[P], q_lo[P];
  int q_scale[P];  // bytes 0, 1: of hi and lo
#pragma unroll
  for (int j = 0; j < P; ++j) {
    int code[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      uint32_t w[8];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint4 v = q_piece(j, b, e);
        w[4 * e] = v.x, w[4 * e + 1] = v.y, w[4 * e + 2] = v.z, w[4 * e + 3] = v.w;
      }
      uint32_t most = 0u;
#pragma unroll
      for (int e = 0; e < 8; ++e) most = max(max(most, (w[e] << 16) & 0x7fffffffu),
                                             w[e] & 0x7fff0000u);
      const auto both = __builtin_amdgcn_permlane32_swap(most, most, false, false);
      const int top = static_cast<int>(max(both[0], both[1]) >> 23);
      code[b] = min(max(top - 7, 6), 254);  // the largest magnitude is in [128, 256)
      const float x_hi = __uint_as_float(static_cast<uint32_t>(code[b]) << 23);
      const float x_lo = __uint_as_float(static_cast<uint32_t>(code[b] - 5) << 23);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        short2_t hi = {0, 0}, lo = {0, 0};
        // lo is what hi's codes leave of q, whichever way they were rounded.
        auto pair = [&](uint32_t whole, auto upper) {
          constexpr bool kUpper = decltype(upper)::value;
          hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(hi, as_pair(whole), x_hi, kUpper);
          const auto held = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(
              __builtin_bit_cast(uint32_t, hi), x_hi, kUpper);
          lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(
              lo, __uint_as_float(whole << 16) - held[0],
              __uint_as_float(whole & 0xffff0000u) - held[1], x_lo, kUpper);
        };
        pair(w[2 * e], std::false_type{});
        pair(w[2 * e + 1], std::true_type{});
        // An infinity or a NaN: the block is NaN.
        q_hi[j][4 * b + e] = top == 255 ? 0x7f7f7f7f : __builtin_bit_cast(int, hi);
        q_lo[j][4 * b + e] = __builtin_bit_cast(int, lo);
      }
    }
    q_scale[j] = half == 0 ? code[0] | (code[0] - 5) << 8 : code[1] | (code[1] - 5) << 8;
  }

  auto qk = [&](const Raw& r) {
    floatx16 s;
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = 0.0f;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const intx8 k = {static_cast<int>(r.c[j][0]), static_cast<int>(r.c[j][1]),
                       static_cast<int>(r.c[j][2]), static_cast<int>(r.c[j][3]), 0, 0, 0, 0};
      const int scale = static_cast<int>(r.s[j]);  // 255: NaN
      s = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(k, q_lo[j], s, 4, 0, 0, scale, 1,
                                                          q_scale[j]);
      s = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(k, q_hi[j], s, 4, 0, 0, scale, 0,
                                                          q_scale[j]);
    }
    return s;
  };
  // The prefix.  This wave's codes two tiles (windows) on are on their way.
  auto products = [&](int t, auto parity) {  // of tile t, whose K is in rk[parity]
    constexpr int p = decltype(parity)::value;
    const floatx16 s = qk(rk[p]);
    if (t + 2 * streams < tiles) load_k(t + 2 * streams, rk[p]);
    return s;
  };
  auto attend = [&](floatx16 x, int t, const unsigned char* v0) {
    const int left = prefix_keys - t * kTileKeys;
    if (left < kTileKeys) mask(x, left, 0xffffu);
    weigh(x, v0);
  };
  using Even = std::integral_constant<int, 0>;
  using Odd = std::integral_constant<int, 1>;
  if constexpr (!kShared) {
    auto step = [&](int t, auto parity) {
      constexpr int p = decltype(parity)::value;
      put_v(rv[p]);
      if (t + 2 * streams < tiles) load_v(t + 2 * streams, rv[p]);
      attend(products(t, parity), t, s_v);
    };
    for (int t = ks; t < tiles; t += 2 * streams) {
      step(t, Even{});
      if (t + streams < tiles) step(t + streams, Odd{});
    }
  } else {
    auto window = [&](int w, auto parity) {
      constexpr int p = decltype(parity)::value;
      __syncthreads();  // stage p is whole, the other one read
      if (w + 1 < windows) {
        if constexpr (kBoth) put_k(rk[1 - p], 1 - p);
        put_w(rv[1 - p], 1 - p);
        if (w + 3 < windows) {
          if constexpr (kBoth) load_kw(w + 3, rk[1 - p]);
          load_v(w + 3, rv[1 - p]);
        }
      }
      const unsigned char* v0 = sh.buf + p * kWindow * ROWB;
      if constexpr (kBoth) {
        if (!active) return;
        attend(qk(take_k(p, 0)), 2 * w, v0);
        if (2 * w + 1 >= tiles) return;
        attend(qk(take_k(p, 1)), 2 * w + 1, v0 + kTileKeys * ROWB);
      } else {
        const int t = 2 * w + ks;
        if (t < tiles) attend(products(t, parity), t, v0 + ks * kTileKeys * ROWB);
      }
    };
    if (windows > 0) {
      if constexpr (kBoth) put_k(rk[0], 0);
      put_w(rv[0], 0);
      if (windows > 2) {
        if constexpr (kBoth) load_kw(2, rk[0]);
        load_v(2, rv[0]);
      }
    }
    for (int w = 0; w < windows; w += 2) {
      window(w, Even{});
      if (w + 1 < windows) window(w + 1, Odd{});
    }
  }

  // st.acc[db][r] holds column 32*db + 8*(r/4) + 4*half + (r%4) of this lane's query.
  if (odd_tiles != 0u) {
    const ArgsIn z = fresh(in);
    const int64_t tree_row_stride = z->attn.tree_row_stride;
    const uint16_t* vt = static_cast<const uint16_t*>(z->attn.v_tree_dev) +
                         g * z->attn.tree_head_stride +
                         static_cast<int64_t>(r0) * tree_row_stride + 4 * half;
    for (int t = 0; t < kAncWords; ++t) {
      if (((odd_tiles >> t) & 1u) == 0u) continue;
      const uint32_t word = sh.anc[r_local][t];
#pragma unroll 1
      for (int j = 0; j < kTileKeys && kTileKeys * t + j < n; ++j) {
        const uint16_t* vr = vt + static_cast<int64_t>(kTileKeys * t + j) * tree_row_stride;
        const bool sees = ((word >> j) & 1u) != 0u;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4) {
            const uint2 v = *reinterpret_cast<const uint2*>(vr + 32 * db + 8 * q4);
            const uint32_t w[2] = {v.x, v.y};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t h = (w[e >> 1] >> (16 * (e & 1))) & 0xffffu;
              if (sees && (h & 0x7f80u) == 0x7f80u)
                st.acc[db][4 * q4 + e] += __uint_as_float(h << 16);
            }
          }
      }
    }
  }
  __syncthreads();

  if constexpr (!kShared) {
    // The states of the q-group's four waves meet in LDS (the V tiles are done with);
    // each of them merges a quarter of the columns and stores it.  (One wave for all of
    // it, through a staging tile, took 4.5 us of a unit, issuing by itself.)
    float* own = reinterpret_cast<float*>(sh.buf + wave * Shared<D>::kSlot);
    own[lane] = st.m;
    own[64 + lane] = st.l;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) own[(2 + 16 * db + r) * 64 + lane] = st.acc[db][r];
    __syncthreads();
    const float* slots =
        reinterpret_cast<const float*>(sh.buf + qg * Shared<D>::kSlot) + lane;
    constexpr int kNext = (kWaves / streams) * Shared<D>::kSlot / 4;  // the next stream's
    float m_all = -__builtin_inff();
#pragma unroll
    for (int k = 0; k < streams; ++k) m_all = fmaxf(m_all, slots[k * kNext]);
    const float m_use = (m_all == -__builtin_inff()) ? 0.0f : m_all;
    float w[streams], l = 0.0f;
#pragma unroll
    for (int k = 0; k < streams; ++k) {
      const float mk = slots[k * kNext];
      w[k] = (mk == -__builtin_inff()) ? 0.0f : __builtin_amdgcn_exp2f((mk - m_use) * c2);
      l += w[k] * slots[k * kNext + 64];
    }
    constexpr int kMine = 16 * DB / streams;  // of the 16 DB values of a lane
    const int first = kMine * ks;
    float o[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      o[i] = 0.0f;
#pragma unroll
      for (int k = 0; k < streams; ++k)
        o[i] += w[k] * slots[k * kNext + (2 + first + i) * 64];
    }
    const ArgsIn z = fresh(in);
    // Values 4 c .. 4 c + 3 of a lane are columns 8 c + 4 half .. + 3 of its query.
    if (u.partial >= 0) {
      // Layout: O as float4 chunks (2 c + half) * 128 + m, then the running max (log2
      // units) and sum per query vector.
      float* part = static_cast<float*>(z->attn.workspace_dev) + partial_floats(D) * u.partial;
#pragma unroll
      for (int c = 0; c < kMine / 4; ++c)
        reinterpret_cast<float4*>(part)[(2 * (first / 4 + c) + half) * kQPerUnit + m] =
            make_float4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
      if (ks == 0 && half == 0) {
        part[static_cast<size_t>(kQPerUnit) * D + m] = (m_all == -__builtin_inff()) ? m_all
                                                                                    : m_all * c2;
        part[static_cast<size_t>(kQPerUnit) * D + kQPerUnit + m] = l;
      }
      return;
    }
    if (r_local >= u.row_count) return;
    const float inv = l > 0.0f ? 1.0f / l : l;  // NaN stays NaN
    uint16_t* dst = static_cast<uint16_t*>(z->attn.out_dev) + row * z->attn.out_row_stride +
                    static_cast<int64_t>(head) * z->attn.out_head_stride + 2 * first + 4 * half;
#pragma unroll
    for (int c = 0; c < kMine / 4; ++c)
      *reinterpret_cast<uint2*>(dst + 8 * c) =
          make_uint2(pack_bf16x2(o[4 * c] * inv, o[4 * c + 1] * inv),
                     pack_bf16x2(o[4 * c + 2] * inv, o[4 * c + 3] * inv));
    return;
  }

  // Merge the key streams of each q-group through LDS (done by one wave each:
  // shared between both as above it measured the same).
  if (active && ks > 0) {
    float* slot = reinterpret_cast<float*>(sh.buf + ((ks - 1) * nq + qg) * Shared<D>::kSlot);
    slot[lane] = st.m;
    slot[64 + lane] = st.l;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) slot[(2 + 16 * db + r) * 64 + lane] = st.acc[db][r];
  }
  __syncthreads();
  if (!active || ks > 0) return;
  for (int k = 1; k < streams; ++k) {
    const float* slot =
        reinterpret_cast<const float*>(sh.buf + ((k - 1) * nq + qg) * Shared<D>::kSlot);
    const float ms = slot[lane];
    const float m_all = fmaxf(st.m, ms);
    const float m_use = (m_all == -__builtin_inff()) ? 0.0f : m_all;
    const float w0 =
        (st.m == -__builtin_inff()) ? 0.0f : __builtin_amdgcn_exp2f((st.m - m_use) * c2);
    const float w1 = (ms == -__builtin_inff()) ? 0.0f : __builtin_amdgcn_exp2f((ms - m_use) * c2);
    st.l = st.l * w0 + w1 * slot[64 + lane];
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        st.acc[db][r] = st.acc[db][r] * w0 + w1 * slot[(2 + 16 * db + r) * 64 + lane];
    st.m = m_all;
  }

  if (u.partial >= 0) {
    // Partial layout (floats): O as float4 chunks ((db*4 + q4)*2 + half)*128 + m,
    // then the running max (log2 units) and sum per query vector.
    float* part = static_cast<float*>(fresh(in)->attn.workspace_dev) + partial_floats(D) * u.partial;
    float4* o = reinterpret_cast<float4*>(part);
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4)
        o[((db * 4 + q4) * 2 + half) * kQPerUnit + m] =
            make_float4(st.acc[db][4 * q4], st.acc[db][4 * q4 + 1], st.acc[db][4 * q4 + 2],
                        st.acc[db][4 * q4 + 3]);
    if (half == 0) {
      part[static_cast<size_t>(kQPerUnit) * D + m] =
          (st.m == -__builtin_inff()) ? st.m : st.m * c2;
      part[static_cast<size_t>(kQPerUnit) * D + kQPerUnit + m] = st.l;
    }
    return;
  }
  // Output through a staging tile of this wave (32 query vectors, rows padded by
  // 16 bytes), behind the merge slots where there are any.
  unsigned char* stage =
      sh.buf + (streams - 1) * nq * Shared<D>::kSlot + qg * Shared<D>::kStage;
  const float inv = st.l > 0.0f ? 1.0f / st.l : st.l;  // NaN stays NaN
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      uint2 packed;
      packed.x = pack_bf16x2(st.acc[db][4 * q4] * inv, st.acc[db][4 * q4 + 1] * inv);
      packed.y = pack_bf16x2(st.acc[db][4 * q4 + 2] * inv, st.acc[db][4 * q4 + 3] * inv);
      *reinterpret_cast<uint2*>(stage + col * kPitch + 2 * (32 * db + 8 * q4 + 4 * half)) =
          packed;
    }
  __builtin_amdgcn_wave_barrier();
  const ArgsIn o = fresh(in);
  const int64_t out_row = o->attn.out_row_stride, out_head = o->attn.out_head_stride;
  uint16_t* const out_base = static_cast<uint16_t*>(o->attn.out_dev) +
                             (static_cast<int64_t>(r0) + u.row_begin) * out_row +
                             static_cast<int64_t>(u.kv_head * G) * out_head;
  auto dst_of = [&](int q, int within) {
    const int mq = qg * 32 + q;
    const int rq = mq >> g_bits;
    return rq < u.row_count
               ? out_base + static_cast<int64_t>(rq) * out_row +
                     static_cast<int64_t>(mq - rq * G) * out_head + within / 2
               : nullptr;
  };
  if (((out_row | out_head) & 7) == 0 &&
      (reinterpret_cast<uintptr_t>(o->attn.out_dev) & 15) == 0) {
#pragma unroll
    for (int i = 0; i < 32 * ROWB / 1024; ++i) {
      const int linear = i * 1024 + 16 * lane;
      const int q = linear / ROWB;
      const int within = linear - q * ROWB;
      const uint4 v = *reinterpret_cast<const uint4*>(stage + q * kPitch + within);
      uint16_t* dst = dst_of(q, within);
      if (dst != nullptr) *reinterpret_cast<uint4*>(dst) = v;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32 * ROWB / 512; ++i) {
      const int linear = i * 512 + 8 * lane;
      const int q = linear / ROWB;
      const int within = linear - q * ROWB;
      const uint2 v = *reinterpret_cast<const uint2*>(stage + q * kPitch + within);
      uint16_t* dst = dst_of(q, within);
      if (dst != nullptr) *reinterpret_cast<uint2*>(dst) = v;
    }
  }
}

// One workgroup per work list (direct: the unit records when every list is one).
template <int D>
__global__ __launch_bounds__(kThreads, 2) void tree_attn_mx4_kernel(SgTreeAttnMx4Args a,
                                                                     const AttnUnit* direct) {
  __shared__ Shared<D> sh;
  const ArgsIn in = (ArgsIn)__builtin_amdgcn_kernarg_segment_ptr();
  const int group = a.attn.num_q_heads / a.attn.num_kv_heads;
  const AttnUnit* units = direct;
  int k = blockIdx.x;
  int end = k + 1;
  if (direct == nullptr) {
    const PlanHeader* hdr = static_cast<const PlanHeader*>(a.attn.plan_dev);
    units = reinterpret_cast<const AttnUnit*>(hdr + 1);
    const int32_t* bin_offset = reinterpret_cast<const int32_t*>(
        reinterpret_cast<const MergeGroup*>(units + hdr->num_units) + hdr->num_merges);
    k = bin_offset[blockIdx.x];
    end = bin_offset[blockIdx.x + 1];
  }
  for (; k < end; ++k) {
    const AttnUnit u = units[k];
    const int vectors = u.row_count * group;
    if (vectors <= 32) {
      attn_unit_mx4<D, false, false>(a, in, u, sh);
    } else if (vectors <= 64) {
      attn_unit_mx4<D, true, false>(a, in, u, sh);
    } else {
      attn_unit_mx4<D, true, true>(a, in, u, sh);
    }
    __syncthreads();  // LDS of this unit is free before the next one starts
  }
}

}  // namespace
}  // namespace sg

namespace sg {
namespace {

// What a unit takes, in microseconds on MI355X: a fixed part (prologue latency, Q's
// terms, the tree, the epilogue) and a part per 64 keys, by its q-groups, with a second
// unit on the CU or alone on it.  Measured over prefixes of 1,024 to 16,384 keys.
struct UnitCost {
  double fixed[2];
  double window[2][4];
};
constexpr UnitCost kCost64 = {{6.0, 4.0}, {{0.49, 0.88, 1.48, 1.50}, {0.33, 0.67, 1.00, 1.03}}};
constexpr UnitCost kCost128 = {{11.0, 7.0}, {{0.88, 1.35, 2.20, 2.33}, {0.63, 0.93, 1.62, 1.74}}};

// The units of a wave by size: `count` of `micros` each.
struct Alike {
  double micros;
  int64_t count;
};

// When the last of the units ends, if they start in decreasing size on `slots` slots.
double end_of(std::vector<Alike>& units, int64_t slots) {
  std::sort(units.begin(), units.end(),
            [](const Alike& a, const Alike& b) { return a.micros > b.micros; });
  std::map<double, int64_t> free;  // time -> slots that become free then
  free[0.0] = slots;
  double end = 0.0;
  for (Alike u : units)
    while (u.count > 0) {
      const auto first = free.begin();
      const double done = first->first + u.micros;
      const int64_t taken = std::min(first->second, u.count);
      u.count -= taken;
      if ((first->second -= taken) == 0) free.erase(first);
      free[done] += taken;
      end = std::max(end, done);
    }
  return end;
}

// A unit in 4 bits takes a third to two thirds of its bf16 time per key but as long for
// what is fixed, and a long one holds the launch's end up as much: prefixes are cut so
// that the estimated end of the last unit, and of the merge that pieces need, is earliest.
// Against the bf16 plan, in turn, 32 q / 8 kv heads, d = 128: 32 requests of 8,192-32,768
// tokens and 1 to 64 rows 432 us (692); 7 of 16,307-32,614 and one row 48 (65); 7 of
// 524-1,048 and 1 to 64 rows 25 (29); 64 of 512-4,096 and 16 to 128 rows 84 (85); d = 64,
// 2 of 27,218 and 256 rows 162 (234).
int plan_mx4(PlanWave wave, const PlanOut& out) {
  if (const int rc = check_plan_wave(wave, out)) return rc;
  const int num_requests = wave.num_requests, num_kv_heads = wave.num_kv_heads;
  const int32_t* const row_offset_host = wave.row_offset;
  const int32_t* const prefix_len_host = wave.prefix_len;
  const int G = wave.num_q_heads / num_kv_heads;
  const int rpt = kQPerUnit / G;
  const UnitCost& cost = wave.head_dim == 64 ? kCost64 : kCost128;
  // A unit of `rows` rows over `keys` keys, and over its request's tree if it is the
  // last piece.
  auto micros = [&](int rows, double keys, int tree_rows, bool alone) {
    const int nq = std::max(1, (rows * G + 31) / 32);
    return cost.fixed[alone] + cost.window[alone][nq - 1] * (keys + tree_rows) / 64.0;
  };
  auto rows_of = [&](int i) { return row_offset_host[i + 1] - row_offset_host[i]; };

  double total = 0.0;
  int64_t whole = 0;
  for (int i = 0; i < num_requests; ++i)
    for (int r = 0; r < rows_of(i); r += rpt) {
      total += num_kv_heads * micros(std::min(rpt, rows_of(i) - r), prefix_len_host[i],
                                     rows_of(i), false);
      whole += num_kv_heads;
    }
  constexpr int64_t kSlots = kDefaultCUs * kListsPerCU;
  const double mean = std::max(1.0, (total - whole * cost.fixed[0]) / kSlots);
  wave.splits.assign(num_requests, 1);
  wave.split_rows.assign(num_requests, 0);
  double best_end = 0.0;
  std::vector<int> splits(num_requests, 1), last_splits;
  std::vector<char> halves(num_requests, 0), last_halves;
  std::vector<Alike> units;
  // Whole units; then those above `share` of a slot's mean load cut by rows, into units
  // of 64 query vectors, which need no merge but pass the keys twice; then by keys, into
  // pieces of at most that load and at least 256 keys.
  struct Cut {
    bool by_rows;
    double share;
  };
  constexpr Cut kCuts[] = {{false, 0.0},  {true, 2.0},  {true, 1.6},
                           {true, 1.4},   {true, 1.2},  {true, 1.0},  {false, 2.0},
                           {false, 1.6},  {false, 1.35}, {false, 1.15}, {false, 1.05}, {false, 0.8},
                           {false, 0.6}, {false, 0.45}, {false, 0.3}};
  for (const Cut& cut : kCuts) {
    int64_t count = 0;
    double partial_bytes = 0.0;
    for (int i = 0; i < num_requests; ++i) {
      const int rows = rows_of(i);
      if (rows == 0) continue;
      const double keys_us =
          micros(std::min(rows, rpt), prefix_len_host[i], 0, false) - cost.fixed[0];
      halves[i] = cut.by_rows && keys_us > cut.share * mean && rows * G > kQPerUnit / 2;
      splits[i] = 1;
      if (!cut.by_rows && cut.share > 0.0)
        splits[i] = static_cast<int>(std::max(1.0, std::min(std::ceil(keys_us / (cut.share * mean)),
                                                            std::floor(prefix_len_host[i] / 256.0))));
      const int of = halves[i] ? rpt / 2 : rpt;
      count += static_cast<int64_t>((rows + of - 1) / of) * splits[i] * num_kv_heads;
      if (splits[i] > 1)
        partial_bytes += 4.0 * (wave.head_dim + 2) * rows * wave.num_q_heads * splits[i];
    }
    if (count > 8 * kSlots && cut.share > 0.0) continue;
    if (splits == last_splits && halves == last_halves) continue;
    last_splits = splits;
    last_halves = halves;
    const bool alone = count <= kDefaultCUs;
    units.clear();
    double load = 0.0;
    for (int i = 0; i < num_requests; ++i) {
      const int of = halves[i] ? rpt / 2 : rpt;
      for (int r = 0; r < rows_of(i); r += of) {
        const int rows = std::min(of, rows_of(i) - r);
        const double keys = static_cast<double>(prefix_len_host[i]) / splits[i];
        units.push_back({micros(rows, keys, rows_of(i), alone), num_kv_heads});
        if (splits[i] > 1)
          units.push_back({micros(rows, keys, 0, alone),
                           static_cast<int64_t>(num_kv_heads) * (splits[i] - 1)});
      }
    }
    double largest = 0.0;
    for (const Alike& u : units) {
      load += u.micros * u.count;
      largest = std::max(largest, u.micros);
    }
    const double merge = partial_bytes > 0.0 ? 12.0 + partial_bytes / 4.5e6 : 0.0;
    // No cut ends before its mean load or its largest unit.
    if (cut.share > 0.0 &&
        merge + (alone ? largest : std::max(load / kSlots, 0.78 * largest)) >= best_end)
      continue;
    // A unit that starts at once and ends last has its CU to itself for the longer part
    // (and older waves issue first): 0.68-0.83 of its time beside another one, measured;
    // with a second turn of units on the slots, 0.84-0.96 of the end at the speed of two.
    // The slots' mean load is passed by up to 0.15, less with smaller units or even loads.
    double end = end_of(units, alone ? kDefaultCUs : kSlots);
    if (!alone && end > 0.0) {
      const double grain = largest / end;
      end = std::max(std::min(end, (1.0 + 0.15 * grain * grain) * load / kSlots),
                     end > 1.001 * largest ? 0.93 * end : 0.78 * end);
    }
    end += merge;
    if (cut.share == 0.0 || end < best_end) {
      best_end = end;
      wave.splits = splits;
      wave.split_rows = halves;
    }
    // Whole units that come this near to an even load leave a cut nothing to gain.
    if (cut.share == 0.0 && end < 1.1 * total / kSlots) break;
  }
  wave.pieces_apart = true;
  wave.unit_cost = [&](int rows, int64_t tiles) {
    return static_cast<int64_t>(100.0 * micros(rows, 32.0 * tiles, 0, false));
  };
  return emit_plan(wave, out);
}

}  // namespace
}  // namespace sg

extern "C" int sg_tree_attn_plan_mx4(int32_t num_requests, const int32_t* row_offset_host,
                                     const int32_t* prefix_len_host, int32_t num_q_heads,
                                     int32_t num_kv_heads, int32_t head_dim, void* plan_host,
                                     size_t plan_capacity_bytes, size_t* plan_bytes,
                                     int32_t* plan_units, int32_t* plan_merges,
                                     size_t* workspace_bytes) {
  using namespace sg;
  clear_error();
  const PlanWave wave = {num_requests, row_offset_host, prefix_len_host,
                         num_q_heads,  num_kv_heads,    head_dim};
  const PlanOut out = {plan_host,  plan_capacity_bytes, plan_bytes,
                       plan_units, plan_merges,         workspace_bytes};
  return guarded([&] { return plan_mx4(wave, out); });
}

extern "C" int sg_tree_attn_mx4_fwd(const SgTreeAttnMx4Args* args, sg_stream_t stream) {
  using namespace sg;
  clear_error();
  SG_REQUIRE(args != nullptr, "null SgTreeAttnMx4Args");
  const SgTreeAttnArgs& a = args->attn;
  AttnCall call;
  if (const int rc = check_attn_call(a, &call)) return rc;
  // The running maximum is one of raw scores.
  SG_REQUIRE(a.scale > 0.0f && std::isfinite(a.scale), "scale must be positive and finite");
  if (a.plan_units == 0) return SG_OK;
  SG_REQUIRE(args->k_scale_dev && args->v_scale_dev, "null device pointer");
  SG_REQUIRE(a.cache_head_stride % 16 == 0 && a.cache_token_stride % 16 == 0 &&
                 ((reinterpret_cast<uintptr_t>(a.k_cache_dev) |
                   reinterpret_cast<uintptr_t>(a.v_cache_dev)) & 15) == 0,
             "codes must be 16-byte aligned, their strides multiples of 16 bytes");
  // Offsets inside a window are 32-bit.
  SG_REQUIRE(a.cache_token_stride >= 0 && a.cache_token_stride < (int64_t{1} << 24) &&
                 args->scale_token_stride >= 0 && args->scale_token_stride < (int64_t{1} << 24),
             "token strides must lie in [0, 2^24) bytes");
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (a.head_dim == 128) {
    tree_attn_mx4_kernel<128><<<dim3(a.plan_units), dim3(kThreads), 0, s>>>(*args, call.direct);
  } else {
    tree_attn_mx4_kernel<64><<<dim3(a.plan_units), dim3(kThreads), 0, s>>>(*args, call.direct);
  }
  SG_LAUNCH_CHECK();
  return launch_attn_merge(a, call.merge_groups, s);
}
