// Packed tree attention over a prefix held in 4 bits (e2m1 codes with a
// power-of-two scale for 32 values of a row; mx4_cache.hip).
//
// Row k of request i attends to request i's cached prefix and to its own tree
// rows that are ancestors of k or k itself, with softmax(q.k * scale) weights;
// plans, units, split partials and their merge are those of tree_attn.hip.  The
// prefix's values are bf16 values, so the products are the bf16 kernel's over
// the unpacked cache.
//
// A window is 64 keys.  Its codes are 9.2 KB (32 KB in bf16): too few bytes to
// keep in LDS as copies in flight, so every thread loads one 16-byte piece of K
// and one of V (32 values, one scale) into registers two windows ahead, unpacks
// them to bf16 (gfx950: two values an instruction, scale included) and writes
// them to the LDS stage that the previous window finished reading.  One barrier
// a window.  Unpacked once for the workgroup: 32 conversions a thread and
// window, where every wave for itself would need 128.
//   S^T = K Q^T and O^T += V^T P^T with v_mfma_f32_32x32x16_bf16, softmax in
//   registers, one query column per lane pair, as in tree_attn.hip.
// The wave's own (bf16) rows come first, while the first windows are loaded.
#include <type_traits>

#include "tree_attn_common.h"

namespace sg {
namespace {

constexpr int kWindow = 64;  // keys of a window: two 32-key blocks
constexpr int kThreads = 256;

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

// LDS of a workgroup: two stages of K and two of V (the merge scratch and the
// output staging after the last window), and the tree's tables.
template <int D>
struct Shared {
  __align__(1024) unsigned char ring[4 * 2 * kTileKeys * D * 2];
  uint32_t anc[kQPerUnit][kAncWords];
  int2 run[kMaxTreeRows];
  uint32_t odd[kAncWords];  // blocks of 32 tree rows with a V that is no number
};

// One unit.  kTwo: of 1-2 q-groups; two waves share one and take a 32-key block of
// each window (key streams, merged at the end).  Otherwise (3-4) a wave takes
// both blocks.
template <int D, bool kTwo>
__device__ __forceinline__ void attn_unit_mx4(const SgTreeAttnMx4Args& args, const AttnUnit& u,
                                              Shared<D>& sh) {
  const SgTreeAttnArgs& a = args.attn;
  constexpr int KB = D / 16;                  // QK^T k-blocks of 16 head dims
  constexpr int DB = D / 32;                  // PV blocks of 32 head dims
  constexpr int ROWB = D * 2;                 // bytes of an LDS row
  constexpr int TILEB = kTileKeys * ROWB;     // bytes of 32 keys of K (or V)
  constexpr int STAGEB = 2 * TILEB;           // bytes of a window of K (or V)
  constexpr int LOADS = D / 64;               // pieces a thread moves per window
  constexpr int STATE = 2 + 16 * DB;          // floats per lane of a WaveState
  constexpr int kSlotBytes = STATE * 64 * 4;
  constexpr int kRowBytes = 2 * D;
  constexpr int kPitch = kRowBytes + 16;
  static_assert(2 * kSlotBytes + 2 * 32 * kPitch <= 4 * STAGEB &&
                    4 * 32 * kPitch <= 4 * STAGEB,
                "merge scratch and output staging must fit the ring");
  unsigned char* const s_ring = sh.ring;
  uint32_t(*const s_anc)[kAncWords] = sh.anc;
  uint32_t* const s_odd = sh.odd;
  unsigned char* const s_k = s_ring;
  unsigned char* const s_v = s_ring + 2 * STAGEB;

  const int G = a.num_q_heads / a.num_kv_heads;
  // Opaque, so that what follows from it is not kept in registers from one unit
  // of a list to the next (83 registers spilled, and a spill's reload waits for
  // the loads in flight).
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
  const int nq = (u.row_count * G + 31) / 32;
  constexpr int streams = kTwo ? 2 : 1;
  const int qg = wave % nq;
  const int ks = wave / nq;
  const bool active = ks < streams;
  const int m = qg * 32 + col;                // query vector inside the unit
  const int r_local = m / G;
  const int head = u.kv_head * G + (m - r_local * G);
  const bool q_valid = active && r_local < u.row_count;
  const int64_t row = static_cast<int64_t>(r0) + u.row_begin + r_local;
  const int g = u.kv_head;
  const bool do_tree = (u.flags & 1) != 0;

  // Pieces of this thread: key row and 32-value block of the window, K or V.
  // A window's base is scalar, a piece's offset one register for K and V.
  constexpr int kBlocks = D / 32;             // 32-value blocks of a row
  const int prefix_keys = u.key_end - u.key_begin;
  const int windows = (prefix_keys + kWindow - 1) / kWindow;
  const int full = prefix_keys / kWindow;
  const int64_t prefix0 = a.prefix_start_dev[u.req] + u.key_begin;
  const int64_t code0 = g * a.cache_head_stride + prefix0 * a.cache_token_stride;
  const int64_t scale0 = g * args.scale_head_stride + prefix0 * args.scale_token_stride;
  const int piece = D == 128 ? tid : tid & 127;
  const int p_row = piece / kBlocks;
  const int p_blk = piece % kBlocks;
  const bool v_wave = wave >= kThreads / 128;  // D = 64: the upper waves move V
  const uint32_t c_lane = p_row * static_cast<uint32_t>(a.cache_token_stride) + 16 * p_blk;
  const uint32_t s_lane = p_row * static_cast<uint32_t>(args.scale_token_stride) + p_blk;
  struct Raw {
    uint4 code[LOADS];
    uint32_t scale[LOADS];
  };
  // Window w of the prefix into registers.  Keys past the range read the last
  // valid one: its score is masked, its probability 0.
  auto load = [&](int w, Raw& r) {
    uint32_t c_off = c_lane, s_off = s_lane;
    if (w >= full) {
      const int key = min(p_row, prefix_keys - 1 - w * kWindow);
      c_off = key * static_cast<uint32_t>(a.cache_token_stride) + 16 * p_blk;
      s_off = key * static_cast<uint32_t>(args.scale_token_stride) + p_blk;
    }
    const int64_t cb = code0 + static_cast<int64_t>(w) * kWindow * a.cache_token_stride;
    const int64_t sb = scale0 + static_cast<int64_t>(w) * kWindow * args.scale_token_stride;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const bool is_v = D == 128 ? i == 1 : v_wave;
      const unsigned char* c =
          static_cast<const unsigned char*>(is_v ? a.v_cache_dev : a.k_cache_dev) + cb;
      const unsigned char* b =
          static_cast<const unsigned char*>(is_v ? args.v_scale_dev : args.k_scale_dev) + sb;
      r.code[i] = *reinterpret_cast<const uint4*>(c + c_off);
      r.scale[i] = b[s_off];
    }
  };
  // LDS offsets of the piece's first 16-byte chunk (of four) in stage 0 of K and
  // V.  The swizzles are XORs of the chunk index, so chunk c is at that ^ 16 c.
  const int k_row = (p_row & 32) + key_slot(p_row & 31);
  const uint32_t k_at = k_row * ROWB + 16 * ((4 * p_blk) ^ swz_k<D>(k_row));
  const uint32_t v_at = p_row * ROWB + 16 * ((4 * p_blk) ^ swz_v<D>(p_row));
  const uint32_t one_at = v_wave ? v_at + 2 * STAGEB : k_at;  // D = 64
  auto piece_at = [&](int i, int c) {
    return s_ring + (D == 128 ? (i == 1 ? (v_at ^ (16 * c)) + 2 * STAGEB : k_at ^ (16 * c))
                              : one_at ^ (16 * c));
  };
  auto unpack = [&](const Raw& r, int stage) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const float s = __uint_as_float(r.scale[i] << 23);  // 255: converts to NaN
      const uint32_t w[4] = {r.code[i].x, r.code[i].y, r.code[i].z, r.code[i].w};
#pragma unroll
      for (int c = 0; c < 4; ++c)
        *reinterpret_cast<uint4*>(piece_at(i, c) + stage * STAGEB) = unpack8(w[c], s);
    }
  };
  // raw[p] holds window w with w & 1 == p.
  Raw raw[2];
  if (windows > 0) load(0, raw[0]);
  if (windows > 1) load(1, raw[1]);

  if (tid < kAncWords) s_odd[tid] = 0u;  // published by the barriers of what follows
  if (do_tree) build_ancestors(a, u, r0, n, sh.run, s_anc);

  // Query operand: lane supplies Q[row, head, 16*kb + 8*half .. +7].
  bf16x8 qf[KB];
  {
    const uint16_t* qp = static_cast<const uint16_t*>(a.q_dev) + row * a.q_row_stride +
                         static_cast<int64_t>(head) * a.q_head_stride + 8 * half;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
      qf[kb] = as_bf16x8(q_valid ? *reinterpret_cast<const uint4*>(qp + 16 * kb) : zero4());
  }

  // LDS read addresses of this lane inside a 32-key block.
  const int gq = lane >> 4;
  const int jj = lane & 15;
  const int rr = jj >> 2;
  const int cc = jj & 3;
  int k_off[KB];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) k_off[kb] = col * ROWB + 16 * ((2 * kb + half) ^ swz_k<D>(col));
  int v_off[DB][2];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int hi = 0; hi < 2; ++hi) {
      const int vrow = 16 * half + 4 * hi + rr;
      const int chunk = 4 * db + 2 * (gq & 1) + (cc >> 1);
      v_off[db][hi] = vrow * ROWB + 16 * (chunk ^ swz_v<D>(vrow)) + 8 * (cc & 1);
    }

  const float c2 = a.scale * kLog2e;
  WaveState<D> st;
  st.m = -__builtin_inff();
  st.l = 0.0f;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) st.acc[db][r] = 0.0f;

  // S^T of the 32-key block at LDS byte `at` of the K stages.
  auto qk = [&](int at) {
    floatx16 s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.0f;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
      s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
          as_bf16x8(*reinterpret_cast<const uint4*>(s_k + at + k_off[kb])), qf[kb], s, 0, 0, 0);
    return s;
  };
  // Online softmax of the block's scores x (masked already): probabilities in x.
  // The reference point st.m moves only when a lane's maximum grew by more than
  // kLazyLog2 in exp2 units (at most 2^kLazyLog2 is exact in bf16 and fp32).
  auto softmax = [&](float (&x)[16]) {
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
  // O^T += V^T P^T over the block at LDS byte `at` of the V stages.
  auto pv = [&](const float (&x)[16], int at) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      bf16x8 pf;
#pragma unroll
      for (int e = 0; e < 8; ++e) pf[e] = static_cast<__bf16>(x[8 * c + e]);
      const unsigned char* vrows = s_v + at + 8 * c * ROWB;
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const short4_t lo =
            __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(vrows + v_off[db][0]));
        const short4_t hi =
            __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(vrows + v_off[db][1]));
        const short8_t v8 = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        st.acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, v8), pf,
                                                             st.acc[db], 0, 0, 0);
      }
    }
  };
  // Both steps of block b of the window in stage `stage`; limit: keys of the
  // block that exist, bits: which of this lane's 16 keys its row sees.
  auto block = [&](const floatx16& s, int at, int limit, uint32_t bits) {
    float x[16];
#pragma unroll
    for (int r = 0; r < 16; ++r)
      x[r] = (16 * half + r < limit && ((bits >> r) & 1u)) ? s[r] : -__builtin_inff();
    softmax(x);
    pv(x, at);
  };

  // The request's own rows, 64 at a time, through stage 0.  Parents precede
  // their children: no row of the unit sees a tree key behind its last row.
  if (do_tree) {
    const int tree_keys = u.row_begin + u.row_count;
    const int64_t tree0 = g * a.tree_head_stride + static_cast<int64_t>(r0) * a.tree_row_stride;
    for (int key0 = 0; key0 < tree_keys; key0 += kWindow) {
      const int key = min(key0 + p_row, n - 1);
      uint4 v[LOADS][4];
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const bool is_v = D == 128 ? i == 1 : v_wave;
        const uint16_t* src = static_cast<const uint16_t*>(is_v ? a.v_tree_dev : a.k_tree_dev) +
                              tree0 + static_cast<int64_t>(key) * a.tree_row_stride + 32 * p_blk;
#pragma unroll
        for (int c = 0; c < 4; ++c) v[i][c] = *reinterpret_cast<const uint4*>(src + 8 * c);
      }
      __syncthreads();  // the stage is free; s_anc is built
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const bool is_v = D == 128 ? i == 1 : v_wave;
        uint32_t any = 0u;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (is_v) {
            // A value that is no number would reach every row of the block
            // through a product with 0: it is added by itself at the end.
            uint32_t w[4] = {v[i][c].x, v[i][c].y, v[i][c].z, v[i][c].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t odd = nonfinite_halves(w[e]);
              any |= odd;
              w[e] &= ~odd;
            }
            v[i][c] = make_uint4(w[0], w[1], w[2], w[3]);
          }
          *reinterpret_cast<uint4*>(piece_at(i, c)) = v[i][c];
        }
        if (any != 0u) s_odd[(key0 + p_row) >> 5] = 1u;
      }
      __syncthreads();
      if (!active) continue;
      for (int b = streams == 2 ? ks : 0; b < (streams == 2 ? ks + 1 : 2); ++b) {
        const int first = key0 + 32 * b;
        if (first >= tree_keys) break;
        block(qk(b * TILEB), b * TILEB, n - first, s_anc[r_local][first >> 5] >> (16 * half));
      }
    }
    __syncthreads();  // stage 0 is free
  }

  // The prefix.  Window w is read from stage w & 1 while window w + 1 is
  // unpacked into the other one and w + 2 and w + 3 are on their way.
  auto whole_block = [&](const floatx16& s, int at) {
    float x[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = s[r];
    softmax(x);
    pv(x, at);
  };
  auto step = [&](int w, auto parity) {
    constexpr int p = decltype(parity)::value;  // w & 1
    __syncthreads();
    if (w + 1 < windows) {
      unpack(raw[1 - p], 1 - p);
      if (w + 3 < windows) load(w + 3, raw[1 - p]);
    }
    if (w == full || !active) return;
    constexpr int at = p * STAGEB;
    if constexpr (kTwo) {
      const int mine = at + ks * TILEB;
      whole_block(qk(mine), mine);
    } else {
      const floatx16 s0 = qk(at);
      const floatx16 s1 = qk(at + TILEB);
      whole_block(s0, at);
      whole_block(s1, at + TILEB);
    }
  };
  if (windows > 0) {
    unpack(raw[0], 0);
    if (windows > 2) load(2, raw[0]);
  }
  for (int w = 0; w < windows; w += 2) {
    step(w, std::integral_constant<int, 0>{});
    if (w + 1 < windows) step(w + 1, std::integral_constant<int, 1>{});
  }
  if (windows > full && active) {  // the last window, of fewer keys
    const int left = prefix_keys - full * kWindow;
    for (int b = streams == 2 ? ks : 0; b < (streams == 2 ? ks + 1 : 2); ++b) {
      const int at = (full & 1) * STAGEB + b * TILEB;
      if (32 * b < left) block(qk(at), at, left - 32 * b, 0xffffu);
    }
  }
  __syncthreads();

  // Merge the key streams of each q-group through LDS (the ring is free now).
  auto merge_slot = [&](int q) { return reinterpret_cast<float*>(s_ring + q * kSlotBytes); };
  if (active && ks > 0) {
    float* slot = merge_slot(qg);
    slot[lane] = st.m;
    slot[64 + lane] = st.l;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) slot[(2 + 16 * db + r) * 64 + lane] = st.acc[db][r];
  }
  __syncthreads();
  if (!active || ks > 0) return;
  if (streams == 2) {
    const float* slot = merge_slot(qg);
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

  // st.acc[db][r] holds head dim 32*db + 8*(r/4) + 4*half + (r%4) of this lane's query.
  if (do_tree) {
    const uint16_t* vt = static_cast<const uint16_t*>(a.v_tree_dev) + g * a.tree_head_stride +
                         static_cast<int64_t>(r0) * a.tree_row_stride + 4 * half;
    for (int t = 0; t < kAncWords; ++t) {
      if (s_odd[t] == 0u) continue;
      const uint32_t word = s_anc[r_local][t];
#pragma unroll 1
      for (int j = 0; j < 32 && 32 * t + j < n; ++j) {
        const uint16_t* vr = vt + static_cast<int64_t>(32 * t + j) * a.tree_row_stride;
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
  if (u.partial >= 0) {
    // Partial layout (floats): O as float4 chunks ((db*4 + q4)*2 + half)*128 + m,
    // then the running max (log2 units) and sum per query vector.
    float* part = static_cast<float*>(a.workspace_dev) + partial_floats(D) * u.partial;
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
      s_ring + (streams == 2 ? 2 * kSlotBytes : 0) + qg * 32 * kPitch;
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
  uint16_t* const out_base = static_cast<uint16_t*>(a.out_dev) +
                             (static_cast<int64_t>(r0) + u.row_begin) * a.out_row_stride +
                             static_cast<int64_t>(u.kv_head * G) * a.out_head_stride;
  auto dst_of = [&](int q, int within) {
    const int mq = qg * 32 + q;
    const int rq = mq / G;
    return rq < u.row_count
               ? out_base + static_cast<int64_t>(rq) * a.out_row_stride +
                     static_cast<int64_t>(mq - rq * G) * a.out_head_stride + within / 2
               : nullptr;
  };
  if (((a.out_row_stride | a.out_head_stride) & 7) == 0 &&
      (reinterpret_cast<uintptr_t>(a.out_dev) & 15) == 0) {
#pragma unroll
    for (int i = 0; i < 32 * kRowBytes / 1024; ++i) {
      const int linear = i * 1024 + 16 * lane;
      const int q = linear / kRowBytes;
      const int within = linear - q * kRowBytes;
      const uint4 v = *reinterpret_cast<const uint4*>(stage + q * kPitch + within);
      uint16_t* dst = dst_of(q, within);
      if (dst != nullptr) *reinterpret_cast<uint4*>(dst) = v;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32 * kRowBytes / 512; ++i) {
      const int linear = i * 512 + 8 * lane;
      const int q = linear / kRowBytes;
      const int within = linear - q * kRowBytes;
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
    if (u.row_count * group <= 64) {
      attn_unit_mx4<D, true>(a, u, sh);
    } else {
      attn_unit_mx4<D, false>(a, u, sh);
    }
    __syncthreads();  // LDS of this unit is free before the next one starts
  }
}

}  // namespace
}  // namespace sg

extern "C" int sg_tree_attn_mx4_fwd(const SgTreeAttnMx4Args* args, sg_stream_t stream) {
  using namespace sg;
  clear_error();
  SG_REQUIRE(args != nullptr, "null SgTreeAttnMx4Args");
  const SgTreeAttnArgs& a = args->attn;
  AttnCall call;
  if (const int rc = check_attn_call(a, &call)) return rc;
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
