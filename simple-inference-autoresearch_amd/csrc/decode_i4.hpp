// Tiles of int4 K/V for decode_main (included by decode_kernel.hpp behind the
// definitions it uses).
//
// Mathematics, for one token's row in groups of G elements:
//   q . k^ = sum_g (s_g sum_{i in g} q_i n_i + m_g sum_{i in g} q_i)
// The first inner sum is one MFMA k-step (or several) on the codes as they
// are: code pairs masked out of a word are fp16 denormals, n 2^-24 or n 2^-20,
// which the matrix cores multiply exactly, so a k-step's 8 codes per lane cost
// five instructions.  s_g is applied to its fp32 result.  The second term, over
// all groups, is one more MFMA: the minima as loaded against the query's sums,
// a fixed operand of the segment, split into two fp16 numbers.
//
// V has its scale along the output's dimension, which no fp32 result can take:
// the values m + n s are formed in fp16, two tokens at a time (n exactly, then
// one rounding), and enter O^T += V^T P^T as 16-bit V does.
//
// Memory: a wave stages its tiles in a ring in LDS, filled by LDS DMA
// (buffer_load ... lds) two tiles ahead and read in operand layout.  A tile of
// head_dim 128 is four transfers of whole rows; loaded straight into registers
// it took 15 narrow loads (64 rows of 16 bytes for K, 4-byte pieces of V and of
// the parameters), and the address unit was busy 73% of a call of 64 x 8192
// tokens, 32/8 heads, that HBM should bound.
//
// Bound: HBM for large calls, closely followed by instruction issue (two waves
// per SIMD, each issuing half of the time); fixed costs for small ones (plan,
// length, page id, first tile, merge: 9 us of the kernel, 3 of the merge
// kernel).  Measured, bf16 queries, the call / the same transfers without the
// arithmetic / the int8 cache:
//   64 x 8192 tokens, 32/8 heads of 128, groups of 64   104 (5.8 TB/s) / 97 / 188 us
//   256 log-normal lengths, 64/8 of 128, groups of 32   220 (5.3 TB/s) / 210 / -
//   32 x 8000, 16/4 of 256, groups of 64                 59 (5.0 TB/s) / 54 / -
//   16 x 0-4096, 16/16 of 64 (fp16), groups of 32        20 / 17 / 45
//   1 x 1000, 32/8 of 128, groups of 64                  12.3 / 9.9 / 13.5
// (The scores of one pair beside V of the pair before, in one wave, took 2.8%
// more: registers, not overlap, are short.)
#pragma once

namespace sia {

template <int D, class KV>
struct I4Tile {
  static constexpr bool kInt8 = false;
  static constexpr int G = KV::group;
  static constexpr int NK = D / G;                        // groups of a row
  static constexpr int NV = D == 256 && G == 32 ? 2 : 1;  // groups that a lane's V share lies in
  static constexpr int NM = NK < 4 ? NK : 4;              // groups per lane of the minima's operand
  static constexpr int KB = D / 8;                        // K bytes per lane: 4 lanes a token
  static constexpr int VB = D / 32;                       // V bytes per lane and token: 16 lanes a token
};
template <int D, class KV>
struct I4K {
  using C = I4Tile<D, KV>;
  Raw<C::KB> k;            // token lane16: word j belongs to k-step j (int4.hpp)
  Raw<4 * C::NM> m;        // token lane16: parameters of groups [4 (grp / 2), +4) (NK = 8), or of all
};
template <int D, class KV>
struct I4KP {
  Raw<4 * I4Tile<D, KV>::NK> t[4];   // tokens 4 grp + i: parameters of every group (step low, minimum high)
};
template <int D, class KV>
struct I4V {
  using C = I4Tile<D, KV>;
  Raw<C::VB> v[4];         // tokens 4 grp + i: codes of the lane's share
  Raw<4 * C::NV> p[4];     // tokens 4 grp + i: parameters of its groups
};

// The ring of one wave: kStages pairs of tiles, a tile K codes, V codes, K parameters, V
// parameters.  Rows of codes are cut into 16-byte pieces, one lane of a
// transfer each:
//  * K rows in token order, the pieces of row r exchanged by r (piece c at
//    place c ^ f(r)), so that 8 lanes reading one piece of 8 tokens touch
//    different banks;
//  * V rows in the order 0, 4, 8, 12, 1, 5, ...: the lanes' shares of tokens
//    4 grp + i (one i, all lanes) are then consecutive.
// Parameters are words in token order.
template <int D, class KV>
struct I4Ring {
  static constexpr int NK = I4Tile<D, KV>::NK;
  static constexpr int RB = D / 2;                        // bytes of a row of codes
  static constexpr int PC = RB / 16;                      // pieces of a row
  static constexpr int KI = D == 256 ? 2 : 1;             // transfers (of 64 pieces) per tensor
  static constexpr int PI = NK == 8 ? 2 : 1;              // transfers (of 64 words) of its parameters
  static constexpr int kV = 1024 * KI, kKP = 2 * kV, kVP = kKP + 256 * PI;
  static constexpr int kTileBytes = kVP + 256 * PI;
  static constexpr int kIds = 2 * kTileBytes;             // ANY: page ids of the pair's tokens, then of the pair again
  static constexpr int kStage = 2 * kTileBytes + (KV::any ? 256 : 0);
  static constexpr int kStages = D == 256 ? 2 : 3;
  static constexpr int kBytes = kStage * kStages;
  static constexpr int kTransfers = 4 * (KI + PI);        // of a stage
  static __device__ __forceinline__ int swizzle(int r) {
    return D == 64 ? (r >> 3) & 1 : D == 128 ? (r >> 2) & 3 : (r >> 1) & 7;
  }
};
// Bytes of LDS per wave: the ring, which also holds the wave's state for the
// merge of a segment (no transfer is then in flight).
template <int D, class KV>
__host__ __device__ constexpr int i4_wave_lds(int G16) {
  return G16 * D * 4 > I4Ring<D, KV>::kBytes ? G16 * D * 4 : I4Ring<D, KV>::kBytes;
}

// A lane's byte offsets: of what it transfers in a tile of the cache (beyond
// any range where it has nothing to), and of what it reads in a stage.
template <int D, class KV>
struct I4Lane {
  using C = I4Tile<D, KV>;
  using R = I4Ring<D, KV>;
  uint32_t k[R::KI], v[R::KI], kp[R::PI];                  // (V's parameters: as K's)
  int rk, rkm, rkp, rv, rvp;
  __device__ __forceinline__ I4Lane(const DecodeArgs& a, int lane) {
    const int lane16 = lane & 15, grp = lane >> 4;
#pragma unroll
    for (int i = 0; i < R::KI; ++i) {
      const int slot = 64 * i + lane, r = slot / R::PC, col = slot % R::PC;
      const bool in = r < kTile;
      k[i] = in ? r * a.k_tok + 16u * (uint32_t)(col ^ R::swizzle(r)) : 0xffffffffu;
      v[i] = in ? (4 * (r & 3) + (r >> 2)) * a.k_tok + 16u * (uint32_t)col : 0xffffffffu;
    }
#pragma unroll
    for (int i = 0; i < R::PI; ++i) {
      const int w = 64 * i + lane, t = w / C::NK, g = w % C::NK;
      kp[i] = t < kTile ? t * a.ks_tok + 4u * (uint32_t)g : 0xffffffffu;
    }
    const int piece = D == 64 ? grp >> 1 : grp;
    rk = lane16 * R::RB + 16 * (piece ^ R::swizzle(lane16)) + (D == 64 ? 8 * (grp & 1) : 0);
    rkm = R::kKP + 4 * C::NK * lane16 + (C::NK == 8 ? 16 * (grp >> 1) : 0);
    rkp = R::kKP + 16 * C::NK * grp;
    rv = R::kV + C::VB * lane;
    rvp = R::kVP + 16 * C::NK * grp + 4 * (8 * i4_word(lane16 * C::VB / 4, D) / C::G);
  }
};

// A tile is transferred through buffer descriptors that end behind its last
// live token: the range check drops the reads behind it (they fill zeros), and
// all of them for the second tile of a pair that has none, so every pair is
// the same number of transfers and every wait a constant.
__device__ __forceinline__ uint32_t i4_range(uint32_t tok, int row, int valid) {
  const uint32_t n = (uint32_t)(min(valid, kTile) - 1) * tok + (uint32_t)row;
  return valid > 0 ? n : 0u;
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t i4_rsrc(const char* p, uint32_t range) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)range, kRawBufferFlags);
}
__device__ __forceinline__ void i4_dma16(__amdgpu_buffer_rsrc_t rs, char* dst, uint32_t off) {
  const int voff = (int)off;
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, dst, 16, voff, 0, 0, kLoadNT);
}
__device__ __forceinline__ void i4_dma4(__amdgpu_buffer_rsrc_t rs, char* dst, uint32_t off) {
  const int voff = (int)off;
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, dst, 4, voff, 0, 0, kLoadNT);
}
template <int D, class KV>
__device__ __forceinline__ void i4_issue(const DecodeArgs& a, const TilePtr& t, const I4Lane<D, KV>& o, int valid,
                                         char* stage) {
  using R = I4Ring<D, KV>;
  const uint32_t codes = i4_range(a.k_tok, R::RB, valid), params = i4_range(a.ks_tok, 4 * R::NK, valid);
  const __amdgpu_buffer_rsrc_t rk = i4_rsrc(t.k, codes), rv = i4_rsrc(t.v, codes);
  const __amdgpu_buffer_rsrc_t rkp = i4_rsrc(t.ks, params), rvp = i4_rsrc(t.vs, params);
#pragma unroll
  for (int i = 0; i < R::KI; ++i) i4_dma16(rk, stage + 1024 * i, o.k[i]);
#pragma unroll
  for (int i = 0; i < R::PI; ++i) i4_dma4(rkp, stage + R::kKP + 256 * i, o.kp[i]);
#pragma unroll
  for (int i = 0; i < R::KI; ++i) i4_dma16(rv, stage + R::kV + 1024 * i, o.v[i]);
#pragma unroll
  for (int i = 0; i < R::PI; ++i) i4_dma4(rvp, stage + R::kVP + 256 * i, o.kp[i]);
}

// ANY: a page holds no whole number of tiles (or one that is no power of two),
// so every token of a tile is looked up.  The page ids of a pair come by a
// transfer of their own, one pair ahead of the rows; lane t + 16 i computes the
// offsets of token t of tile i once, and the lanes that transfer pieces of that
// token's row fetch them from it.  Offsets are 32-bit, from the pool's start.
// 32 sequences of 100-4000 tokens in pages of 24, 32/8 heads of 128: 30.6 us, on
// the vector ALU 251.  (Pages of 16 taken this way cost 1.3% more, over 22
// shapes, than with one page id per tile.)
template <int D, class KV>
struct I4Rows {
  using C = I4Tile<D, KV>;
  using R = I4Ring<D, KV>;
  int k[R::KI], v[R::KI], p[R::PI];            // 4 x the token whose row a lane transfers a piece of
  uint32_t kc[R::KI], vc[R::KI], pc[R::PI];    // that piece's byte in the row; ~0, past every range, for no piece
  __device__ __forceinline__ explicit I4Rows(int lane) {
#pragma unroll
    for (int i = 0; i < R::KI; ++i) {
      const int slot = 64 * i + lane, r = slot / R::PC, col = slot % R::PC, t = r & 15;
      k[i] = 4 * t;
      v[i] = 4 * (4 * (t & 3) + (t >> 2));
      kc[i] = r < kTile ? 16u * (uint32_t)(col ^ R::swizzle(r)) : ~0u;
      vc[i] = r < kTile ? 16u * (uint32_t)col : ~0u;
    }
#pragma unroll
    for (int i = 0; i < R::PI; ++i) {
      const int w = 64 * i + lane, t = w / C::NK;
      p[i] = 4 * (t & 15);
      pc[i] = t < kTile ? 4u * (uint32_t)(w % C::NK) : ~0u;
    }
  }
};
// Tile i of a pair, from the lanes' offsets of rows of codes and parameters.
template <int D, class KV>
__device__ __forceinline__ void i4_issue_rows(__amdgpu_buffer_rsrc_t rk, __amdgpu_buffer_rsrc_t rv,
                                              __amdgpu_buffer_rsrc_t rkp, __amdgpu_buffer_rsrc_t rvp,
                                              const I4Rows<D, KV>& o, int i, uint32_t codes, uint32_t params,
                                              char* stage) {
  using R = I4Ring<D, KV>;
  char* dst = stage + i * R::kTileBytes;
  auto at = [&](uint32_t off, int token, uint32_t byte) {
    const uint32_t row = (uint32_t)__builtin_amdgcn_ds_bpermute(token + 64 * i, (int)off);
    return __builtin_elementwise_add_sat(row, byte);
  };
#pragma unroll
  for (int x = 0; x < R::KI; ++x) i4_dma16(rk, dst + 1024 * x, at(codes, o.k[x], o.kc[x]));
#pragma unroll
  for (int x = 0; x < R::PI; ++x) {
    const uint32_t off = at(params, o.p[x], o.pc[x]);
    i4_dma4(rkp, dst + R::kKP + 256 * x, off);
    i4_dma4(rvp, dst + R::kVP + 256 * x, off);
  }
#pragma unroll
  for (int x = 0; x < R::KI; ++x) i4_dma16(rv, dst + R::kV + 1024 * x, at(codes, o.v[x], o.vc[x]));
}

// At most N of the wave's vector memory instructions still outstanding.
template <int N>
__device__ __forceinline__ void i4_wait() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | ((N >> 4) << 14));
}

template <int BYTES>
__device__ __forceinline__ void i4_read(Raw<BYTES>& r, const char* p) {
  if constexpr (BYTES % 16 == 0) {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const u32x4 x = *(const u32x4*)(p + 16 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) r.w[4 * i + j] = x[j];
    }
  } else if constexpr (BYTES == 8) {
    const u32x2 x = *(const u32x2*)p;
    r.w[0] = x[0];
    r.w[1] = x[1];
  } else if constexpr (BYTES == 4) {
    r.w[0] = *(const uint32_t*)p;
  } else {
    static_assert(BYTES == 2, "tile operand size");
    r.w[0] = *(const uint16_t*)p;
  }
}
template <int D, class KV>
__device__ __forceinline__ void i4_read_k(const char* tile, const I4Lane<D, KV>& o, I4K<D, KV>& c) {
  using C = I4Tile<D, KV>;
  if constexpr (D == 256) {     // pieces grp and grp + 4
    const u32x4 x = *(const u32x4*)(tile + o.rk), y = *(const u32x4*)(tile + (o.rk ^ 64));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      c.k.w[j] = x[j];
      c.k.w[4 + j] = y[j];
    }
  } else {
    i4_read<C::KB>(c.k, tile + o.rk);
  }
  if constexpr (C::NK > 1) i4_read<4 * C::NM>(c.m, tile + o.rkm);
}
template <int D, class KV>
__device__ __forceinline__ void i4_read_kp(const char* tile, const I4Lane<D, KV>& o, I4KP<D, KV>& c) {
  using C = I4Tile<D, KV>;
#pragma unroll
  for (int i = 0; i < 4; ++i) i4_read<4 * C::NK>(c.t[i], tile + o.rkp + 4 * C::NK * i);
}
template <int D, class KV>
__device__ __forceinline__ void i4_read_v(const char* tile, const I4Lane<D, KV>& o, I4V<D, KV>& c) {
  using C = I4Tile<D, KV>;
#pragma unroll
  for (int i = 0; i < 4; ++i) i4_read<C::VB>(c.v[i], tile + o.rv + 64 * C::VB * i);
#pragma unroll
  for (int i = 0; i < 4; ++i) i4_read<4 * C::NV>(c.p[i], tile + o.rvp + 4 * C::NK * i);
}

// The query of a unit: its MFMA operands, its sums over the groups and the
// multiplier of a score.
//
// HALF: at most 8 heads, so the 16 columns hold them twice, and column c + 8
// is head c for the second tile of a pair.  With the query zero in the other
// tile's columns (op[0], op[1]), both tiles accumulate into one result, and the
// softmax of a pair costs what that of one tile did.  (Head_dim 256 has no
// registers for two operands and selects between two results.)
template <int D, class KV>
struct I4Query {
  static constexpr int N = KV::half && D <= 128 ? 2 : 1;
  // |sum| <= 128 x 2^14 in fp16's range, and far above its denormals: the two
  // parts hold 22 bits of it.  (With the codes' 2^-24, which needs no product
  // to join the two, the lower part ends at 2^-14 of the largest |q|, times m.)
  static constexpr float kSums = 0x1p-6f;
  u32x4 op[N][D / 32];
  u32x2 sums[N];  // NK > 1: operand of the minima's product, kSums times the sums in two fp16 parts
  float sum;      // NK = 1: 2^-24 times the sum
  float mul;
};
template <int D, class KV, class QT>
__device__ __forceinline__ void i4_prep_q(const DecodeArgs& a, QRaw<D>& raw, int lane16, int grp, I4Query<D, KV>& q) {
  constexpr int NK = I4Tile<D, KV>::NK, STEPS = D / 32, PER = STEPS / NK;
  // a power of two brings max |q| into [2^13, 2^14): fp16 operands without
  // overflow that lose bits only below 2^-24 of the maximum
  float amax = 0.f;
#pragma unroll
  for (int j = 0; j < STEPS; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      amax = fmaxf(amax, fmaxf(fabsf(lo_f32(QT{}, raw.w[j][i])), fabsf(hi_f32(QT{}, raw.w[j][i]))));
      // (converted again below: kept, the row in fp32 takes D / 4 registers
      // beside the first tile's, more than 4 waves per SIMD leave)
      asm("" : "+v"(raw.w[j][i]));
    }
  amax = wave_max_xor16_32(amax);
  const int sh = amax > 0.f ? 14 - __builtin_amdgcn_frexp_expf(amax) : 0;
  // (2^100 for queries beyond 2^93: with more the score of two different keys
  // differs by far more than the softmax resolves, and the multiplier overflows)
  q.mul = fminf(ldexpf(a.qk_scale, 24 - sh), 0x1p100f);
  float sum[NK];
#pragma unroll
  for (int j = 0; j < STEPS; ++j) {
    float x[8];
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t w = raw.w[j][i >> 1];
      x[i] = ldexpf((i & 1) ? hi_f32(QT{}, w) : lo_f32(QT{}, w), sh);
      t += x[i];
    }
    sum[j / PER] = j % PER == 0 ? t : sum[j / PER] + t;
    // the order and the powers of two of the code pairs (i4_scores)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float f = (i & 1) ? 0.0625f : 1.0f;
      q.op[0][j][i] = pack2(F16{}, x[i] * f, x[i + 4] * f);
    }
  }
#pragma unroll
  for (int g = 0; g < NK; ++g) sum[g] = wave_sum_xor16_32(sum[g]) * (NK == 1 ? 0x1p-24f : I4Query<D, KV>::kSums);
  if constexpr (NK == 1) {
    q.sum = sum[0];
  } else {
    // contraction index 4 grp + i: group i (NK = 8: and 4 more for the upper
    // two lane groups), the high parts in even lane groups, the rest in odd ones
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float f = i < NK ? sum[i < NK ? i : 0] : 0.f;
      if constexpr (NK == 8) f = grp >= 2 ? sum[4 + i] : f;
      else f = grp >= 2 ? 0.f : f;
      const float hi = (float)(_Float16)f;
      x[i] = (grp & 1) ? f - hi : hi;
    }
    q.sums[0] = u32x2{pack2(F16{}, x[0], x[1]), pack2(F16{}, x[2], x[3])};
  }
  if constexpr (I4Query<D, KV>::N == 2) {
    const uint32_t first = lane16 < 8 ? ~0u : 0u;
#pragma unroll
    for (int j = 0; j < STEPS; ++j) {
      q.op[1][j] = q.op[0][j] & ~first;
      q.op[0][j] &= first;
    }
    if constexpr (NK > 1) {
      q.sums[1] = q.sums[0] & ~first;
      q.sums[0] &= first;
    }
  }
}

// acc + K Q over group g's k-steps of one tile.
template <int D, class KV>
__device__ __forceinline__ f32x4 i4_qk(const I4K<D, KV>& c, const u32x4* op, int g, f32x4 acc) {
  constexpr int PER = KV::group / 32;
#pragma unroll
  for (int j = PER * g; j < PER * (g + 1); ++j) {
    // codes (0, 4), (1, 5), (2, 6), (3, 7)
    const uint32_t w = c.k.w[j], w8 = w >> 8;
    const u32x4 ka = {w & 0x000f000fu, w & 0x00f000f0u, w8 & 0x000f000fu, w8 & 0x00f000f0u};
    acc = mfma16x16x32(F16{}, ka, op[j], acc);
  }
  return acc;
}
// acc + the minima's product of one tile.
template <int D, class KV>
__device__ __forceinline__ f32x4 i4_qm(const I4K<D, KV>& c, u32x2 sums, f32x4 acc) {
  constexpr int NM = I4Tile<D, KV>::NM;
  const u32x2 ma = {gather16(c.m.w[0], c.m.w[NM > 1 ? 1 : 0], 1),
                    NM == 4 ? gather16(c.m.w[NM == 4 ? 2 : 0], c.m.w[NM == 4 ? 3 : 0], 1) : 0u};
  return mfma16x16x16(F16{}, ma, sums, acc);
}
// Scores of tokens 4 grp + i, before the multiplier: HALF, of the tile whose
// columns the lane is in (kp: that tile's parameters), else of tile `t`.
template <int D, class KV>
__device__ __forceinline__ void i4_scores(const I4K<D, KV>* c, int t, const I4KP<D, KV>& kp, const I4Query<D, KV>& q,
                                          int lane16, float (&s)[4]) {
  constexpr int NK = I4Tile<D, KV>::NK;
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  // x(tile, operand, start): one tile's product added to `start`
  auto both = [&](auto&& x) -> f32x4 {
    if constexpr (!KV::half) return x(t, 0, zero);
    else if constexpr (I4Query<D, KV>::N == 2) return x(1, 1, x(0, 0, zero));
    else {
      const f32x4 u = x(0, 0, zero), v = x(1, 0, zero);
      return lane16 < 8 ? u : v;
    }
  };
#pragma unroll
  for (int g = 0; g < NK; ++g) {
    const f32x4 acc = both([&](int ti, int qi, f32x4 a0) { return i4_qk<D, KV>(c[ti], q.op[qi], g, a0); });
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float step = lo_f32(F16{}, kp.t[i].w[g]);
      s[i] = g == 0 ? step * acc[i] : __builtin_fmaf(step, acc[i], s[i]);
    }
  }
  if constexpr (NK > 1) {
    const f32x4 z = both([&](int ti, int qi, f32x4 acc) { return i4_qm<D, KV>(c[ti], q.sums[qi], acc); });
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = __builtin_fmaf(z[i], 0x1p-24f / I4Query<D, KV>::kSums, s[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = __builtin_fmaf(hi_f32(F16{}, kp.t[i].w[0]), q.sum, s[i]);
  }
}

// s mul - m with s mul rounded, as the maximum is: never above the threshold,
// however large the scores.  (In one fma the largest score itself is off by
// what the maximum's rounding took, from 2^31 on more than an exponent holds.)
__device__ __forceinline__ float i4_above(float s, float mul, float m) {
#pragma clang fp contract(off)
  const float x = s * mul;
  return x - m;
}

// The weights of 16-bit queries enter the matrix cores in fp16.  Their
// reference st.m stands kI4Lift below the running maximum when that moves, and
// a score moves it from kI4Lazy above on, so that the largest weight is 2^11 to
// 2^15.  One of w times the largest is then rounded by at most 2^-11 w + 2^-36.
// (With the maximum itself for reference the second term is 2^-25: tokens
// behind a sink, each 2^-20 of its weight, came out up to 3% off.)
constexpr float kI4Lift = 11.0f, kI4Lazy = 4.0f;

// Online softmax of NS x 4 scores per lane: weights p (the running maximum
// moves lazily, as in compute_tile).  A score of -inf weighs 0, also before any
// other was seen.  The threshold is compared with the difference, which is exact
// where it matters: a sum st.m + 8 rounds up to st.m + 16 from 2^27 on, and a
// weight of 2^16 is an infinity in fp16.  LIFTED: p goes into fp16 (a reference
// that the subtraction rounds further down stays at the maximum).
template <int D, int NS, bool LIFTED>
__device__ __forceinline__ void i4_softmax(const float (&s)[NS][4], float mul, bool masked, WaveState<D>& st,
                                           float (&p)[NS][4]) {
  constexpr float kMost = LIFTED ? kI4Lift + kI4Lazy : kLazyMax;
  float lmax = -INFINITY;
#pragma unroll
  for (int n = 0; n < NS; ++n) lmax = fmaxf(lmax, fmaxf(fmaxf(s[n][0], s[n][1]), fmaxf(s[n][2], s[n][3])));
  lmax *= mul;
  if (__any(lmax - st.m > kMost)) {
    float ref = wave_max_xor16_32(lmax);
    if constexpr (LIFTED) {
      const float low = ref - kI4Lift;
      ref = ref - low > kMost ? ref : low;
    }
    const float m_new = fmaxf(st.m, ref);
    const float alpha = fast_exp2(st.m - (m_new == -INFINITY ? 0.f : m_new));
    st.m = m_new;
    st.l *= alpha;
#pragma unroll
    for (int e = 0; e < D / 16; ++e) st.acc[e] *= alpha;
  }
#pragma unroll
  for (int n = 0; n < NS; ++n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[n][i] = fast_exp2(i4_above(s[n][i], mul, st.m));
    if (masked) {                  // (uniform)
#pragma unroll
      for (int i = 0; i < 4; ++i) p[n][i] = s[n][i] == -INFINITY ? 0.f : p[n][i];
    }
    st.l += (p[n][0] + p[n][1]) + (p[n][2] + p[n][3]);
  }
}

// Constants of the conversion, in registers: v_and_or_b32 takes no literal
// (as two instructions with a literal each, V cost 16 more per tile).
struct I4Const {
  uint32_t lo, hi;      // masks of the pairs at bits 0-3 and 4-7 of the halves (scalar)
  uint32_t blo, bhi;    // 0x6400 | n is 1024 + n in fp16, 0x5400 | n << 4 is 64 + n
  __device__ __forceinline__ I4Const() {
    asm("s_mov_b32 %0, 0x000f000f" : "=s"(lo));
    asm("s_mov_b32 %0, 0x00f000f0" : "=s"(hi));
    asm("v_mov_b32 %0, 0x64006400" : "=v"(blo));
    asm("v_mov_b32 %0, 0x54005400" : "=v"(bhi));
  }
};

// O^T += V^T P^T over a pair of tiles.  d-tile e takes code e of every lane's
// share, for tokens (4 grp, 4 grp + 1) and (4 grp + 2, 4 grp + 3) of either
// tile.  pop: P in the same order, zero (HALF) in the other tile's columns.
template <int D, class KV>
__device__ __forceinline__ void i4_pv(const I4V<D, KV>* c, const I4Const& ic, u32x4 pop, WaveState<D>& st) {
  using C = I4Tile<D, KV>;
#pragma unroll
  for (int h = 0; h < D / 64; ++h) {        // 4 codes of each token
    const int gv = C::NV == 2 ? h >> 1 : 0;
    uint32_t x[4], x8[4];
    f16x2 s[4], m[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const I4V<D, KV>& v = c[t >> 1];
      const int k = 2 * (t & 1);
      x[t] = gather16(v.v[k].w[h >> 1], v.v[k + 1].w[h >> 1], h & 1);
      x8[t] = x[t] >> 8;
      s[t] = __builtin_bit_cast(f16x2, gather16(v.p[k].w[gv], v.p[k + 1].w[gv], 0));
      m[t] = __builtin_bit_cast(f16x2, gather16(v.p[k].w[gv], v.p[k + 1].w[gv], 1));
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      u32x4 va;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const uint32_t w = e & 2 ? x8[t] : x[t];
        const _Float16 b = e & 1 ? (_Float16)-64.0f : (_Float16)-1024.0f;
        const uint32_t biased = e & 1 ? ((w & ic.hi) | ic.bhi) : ((w & ic.lo) | ic.blo);
        const f16x2 n = __builtin_bit_cast(f16x2, biased) + f16x2{b, b};
        va[t] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(n, s[t], m[t]));
      }
      st.acc[4 * h + e] = mfma16x16x32(F16{}, va, pop, st.acc[4 * h + e]);
    }
  }
}

// One pair of tiles: left0, left1 live tokens.
template <int D, class KV>
__device__ __forceinline__ void i4_pair(const char* stage, const I4Lane<D, KV>& o, const I4Const& ic,
                                        const I4Query<D, KV>& q, int left0, int left1, int lane16, int grp,
                                        WaveState<D>& st) {
  using R = I4Ring<D, KV>;
  constexpr int NS = KV::half ? 1 : 2;
  const bool masked = left0 < kTile || left1 < kTile;
  float s[NS][4], p[NS][4];
  {
    I4K<D, KV> k[2];
    i4_read_k<D, KV>(stage, o, k[0]);
    i4_read_k<D, KV>(stage + R::kTileBytes, o, k[1]);
    if constexpr (I4Query<D, KV>::N == 2 && I4Tile<D, KV>::NK > 1) {
      if (masked) {      // (uniform) one result holds both tiles: 0 x m has to be 0 in a dead token's row
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (lane16 >= (t == 0 ? left0 : left1)) {
#pragma unroll
            for (int g = 0; g < I4Tile<D, KV>::NM; ++g) k[t].m.w[g] = 0u;
          }
      }
    }
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      I4KP<D, KV> kp;
      i4_read_kp<D, KV>(stage + (KV::half ? (lane16 < 8 ? 0 : R::kTileBytes) : n * R::kTileBytes), o, kp);
      i4_scores<D, KV>(k, n, kp, q, lane16, s[n]);
    }
  }
  I4V<D, KV> v[2];
  i4_read_v<D, KV>(stage, o, v[0]);
  i4_read_v<D, KV>(stage + R::kTileBytes, o, v[1]);
  if (masked) {
    // (uniform) the wave's last pair.  Dead tokens weigh 0; their parameters
    // are cleared too, so that the result never depends on what a dropped
    // transfer leaves behind.
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int live = KV::half ? (lane16 < 8 ? left0 : left1) : n == 0 ? left0 : left1;
        if (4 * grp + i >= live) s[n][i] = -INFINITY;
      }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (4 * grp + i >= (t == 0 ? left0 : left1)) {
#pragma unroll
          for (int g = 0; g < I4Tile<D, KV>::NV; ++g) v[t].p[i].w[g] = 0u;
        }
  }
  i4_softmax<D, NS, true>(s, q.mul, masked, st, p);
  u32x4 pop;
  if constexpr (KV::half) {
    const u32x2 w = {pack2(F16{}, p[0][0], p[0][1]), pack2(F16{}, p[0][2], p[0][3])};
    const uint32_t first = lane16 < 8 ? ~0u : 0u;
    pop = u32x4{w[0] & first, w[1] & first, w[0] & ~first, w[1] & ~first};
  } else {
    pop = u32x4{pack2(F16{}, p[0][0], p[0][1]), pack2(F16{}, p[0][2], p[0][3]),
                pack2(F16{}, p[NS - 1][0], p[NS - 1][1]), pack2(F16{}, p[NS - 1][2], p[NS - 1][3])};
  }
  i4_pv<D, KV>(v, ic, pop, st);
}

// ---- fp32 queries: fp32 MFMAs over the values m + n s, each rounded once to fp32
// as kv_read rounds them; nothing is rounded to fewer bits.  Tiles, rings and
// softmax are the same.  Bound: the matrix cores (256 FLOP per cycle per CU, and
// 16 columns whatever the heads): 32 sequences of 100-4000 tokens, 32/8 heads of
// 128, 76 us, on the vector ALU 207.  (Which one: f32_matrix in capi_decode.cpp.)

// A lane's query elements, in the order of its codes of K.
template <int D>
struct I4Query32 {
  f32x4 x[D / 16];
};
template <int D>
__device__ __forceinline__ I4Query32<D> i4_load_q32(const DecodeArgs& a, int b, int hq, bool live, int grp) {
  I4Query32<D> q;
  const char* qp = a.q + b * a.q_sb + (int64_t)hq * a.q_sh + grp * 32;
#pragma unroll
  for (int j = 0; j < D / 16; ++j)
    q.x[j] = live ? *(const f32x4*)(qp + 128 * (j >> 1) + 16 * (j & 1)) : f32x4{0.f, 0.f, 0.f, 0.f};
  return q;
}
__device__ __forceinline__ f32x4 i4_mfma32(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
// Value i of a word of codes (even: the codes at bits 0-3 of the bytes, odd: at 4-7).
__device__ __forceinline__ float i4_value_of(uint32_t even, uint32_t odd, int i, uint32_t sm) {
  const uint32_t w = (i & 1) ? odd : even;
  const float n = (float)(uint8_t)(w >> (8 * (i >> 1)));
  return __builtin_fmaf(n, lo_f32(F16{}, sm), hi_f32(F16{}, sm));
}
template <int D, class KV>
__device__ __forceinline__ void i4_pair32(const char* stage, const I4Lane<D, KV>& o, const I4Query32<D>& q, float mul,
                                          int left0, int left1, int lane16, int grp, WaveState<D>& st) {
  using R = I4Ring<D, KV>;
  using C = I4Tile<D, KV>;
  constexpr int PER = C::G / 32;
  const bool masked = left0 < kTile || left1 < kTile;
  float s[2][4], p[2][4];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const char* tile = stage + t * R::kTileBytes;
    I4K<D, KV> k;
    i4_read_k<D, KV>(tile, o, k);
    Raw<4 * C::NK> sm;                                        // of the lane's token
    i4_read<4 * C::NK>(sm, tile + R::kKP + 4 * C::NK * lane16);
    f32x4 acc[2] = {};                                        // (two chains: half the roundings of one)
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      const uint32_t even = k.k.w[j] & 0x0f0f0f0fu, odd = (k.k.w[j] >> 4) & 0x0f0f0f0fu;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        acc[i & 1] = i4_mfma32(i4_value_of(even, odd, i, sm.w[j / PER]), q.x[2 * j + (i >> 2)][i & 3], acc[i & 1]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) s[t][i] = acc[0][i] + acc[1][i];
  }
  I4V<D, KV> v[2];
  i4_read_v<D, KV>(stage, o, v[0]);
  i4_read_v<D, KV>(stage + R::kTileBytes, o, v[1]);
  if (masked) {      // (uniform) as in i4_pair
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (4 * grp + i >= (t == 0 ? left0 : left1)) {
          s[t][i] = -INFINITY;
#pragma unroll
          for (int g = 0; g < C::NV; ++g) v[t].p[i].w[g] = 0u;
        }
  }
  i4_softmax<D, 2, false>(s, mul, masked, st, p);
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int h = 0; h < D / 128 + (D == 64); ++h) {         // words of the lane's share (D = 64: half of one)
        const uint32_t w = v[t].v[i].w[h], even = w & 0x0f0f0f0fu, odd = (w >> 4) & 0x0f0f0f0fu;
        const uint32_t sm = v[t].p[i].w[C::NV == 2 ? h : 0];
#pragma unroll
        for (int e = 0; e < (D == 64 ? 4 : 8); ++e)
          st.acc[8 * h + e] = i4_mfma32(i4_value_of(even, odd, e, sm), p[t][i], st.acc[8 * h + e]);
      }
}

// HALF: the two tiles' states of a head, columns c and c + 8, added up.
template <int D>
__device__ __forceinline__ void i4_join(WaveState<D>& st) {
  auto other = [](float x) {      // of lane16 ^ 8: a rotation by 8 inside each row of 16 lanes
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x128, 0xf, 0xf, false));
  };
  const float m = fmaxf(st.m, other(st.m));
  const float w = fast_exp2(st.m - (m == -INFINITY ? 0.f : m));
  st.m = m;
  st.l *= w;
  st.l += other(st.l);
#pragma unroll
  for (int e = 0; e < D / 16; ++e)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = st.acc[e][i] * w;
      st.acc[e][i] = x + other(x);
    }
}

}  // namespace sia
