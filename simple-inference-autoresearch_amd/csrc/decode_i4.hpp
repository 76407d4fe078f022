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
  Raw<KB> k;               // token lane16: word j belongs to k-step j (int4.hpp)
  Raw<4 * NM> km;          // token lane16: parameters of groups [4 (grp / 2), +4) (NK = 8), or of all
  Raw<4 * NK> kp[4];       // tokens 4 grp + i: parameters of every group (step low, minimum high)
  Raw<VB> v[4];            // tokens 4 grp + i: codes of the lane's share
  Raw<4 * NV> vp[4];       // tokens 4 grp + i: parameters of its groups
};

// The ring of one wave: kStages tiles, each K codes, V codes, K parameters, V
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
  static constexpr int kStage = kVP + 256 * PI;
  static constexpr int kStages = 3;
  static constexpr int kBytes = kStage * kStages;
  static constexpr int kTransfers = 2 * (KI + PI);        // of a tile
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
// live token: the range check drops the reads behind it (they fill zeros) and,
// for a tile without live tokens (behind a wave's last one), all of them, so
// every round of the loop issues the same number of transfers and its wait is
// a constant.
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
__device__ __forceinline__ void i4_read_k(const char* stage, const I4Lane<D, KV>& o, I4Tile<D, KV>& c) {
  using C = I4Tile<D, KV>;
  if constexpr (D == 256) {     // pieces grp and grp + 4
    const u32x4 x = *(const u32x4*)(stage + o.rk), y = *(const u32x4*)(stage + (o.rk ^ 64));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      c.k.w[j] = x[j];
      c.k.w[4 + j] = y[j];
    }
  } else {
    i4_read<C::KB>(c.k, stage + o.rk);
  }
  if constexpr (C::NK > 1) i4_read<4 * C::NM>(c.km, stage + o.rkm);
#pragma unroll
  for (int i = 0; i < 4; ++i) i4_read<4 * C::NK>(c.kp[i], stage + o.rkp + 4 * C::NK * i);
}
template <int D, class KV>
__device__ __forceinline__ void i4_read_v(const char* stage, const I4Lane<D, KV>& o, I4Tile<D, KV>& c) {
  using C = I4Tile<D, KV>;
#pragma unroll
  for (int i = 0; i < 4; ++i) i4_read<C::VB>(c.v[i], stage + o.rv + 64 * C::VB * i);
#pragma unroll
  for (int i = 0; i < 4; ++i) i4_read<4 * C::NV>(c.vp[i], stage + o.rvp + 4 * C::NK * i);
}

// The query of a unit: its MFMA operands, its sums over the groups and the
// multiplier of a score.
template <int D, class KV>
struct I4Query {
  u32x4 op[D / 32];
  u32x2 sums;     // NK > 1: operand of the minima's product, 2^-24 times the sums in two fp16 parts
  float sum;      // NK = 1: 2^-24 times the sum
  float mul;
};
template <int D, class KV, class QT>
__device__ __forceinline__ void i4_prep_q(const DecodeArgs& a, QRaw<D>& raw, int grp, I4Query<D, KV>& q) {
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
  q.mul = ldexpf(a.qk_scale, 24 - sh);
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
      q.op[j][i] = pack2(F16{}, x[i] * f, x[i + 4] * f);
    }
  }
#pragma unroll
  for (int g = 0; g < NK; ++g) sum[g] = wave_sum_xor16_32(sum[g]) * 0x1p-24f;
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
    q.sums = u32x2{pack2(F16{}, x[0], x[1]), pack2(F16{}, x[2], x[3])};
  }
}

// Scores of tokens 4 grp + i for head lane16, before the multiplier.
template <int D, class KV>
__device__ __forceinline__ void i4_scores(const I4Tile<D, KV>& c, const I4Query<D, KV>& q, float (&s)[4]) {
  constexpr int NK = I4Tile<D, KV>::NK, PER = KV::group / 32;
  f32x4 t = {0.f, 0.f, 0.f, 0.f};
  if constexpr (NK > 1) {
    constexpr int NM = I4Tile<D, KV>::NM;
    const u32x2 ma = {gather16(c.km.w[0], c.km.w[1], 1), NM == 4 ? gather16(c.km.w[NM - 2], c.km.w[NM - 1], 1) : 0u};
    t = mfma16x16x16(F16{}, ma, q.sums, t);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) s[i] = NK == 1 ? hi_f32(F16{}, c.kp[i].w[0]) * q.sum : t[i];
#pragma unroll
  for (int g = 0; g < NK; ++g) {
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = PER * g; j < PER * (g + 1); ++j) {
      // codes (0, 4), (1, 5), (2, 6), (3, 7)
      const uint32_t w = c.k.w[j], w8 = w >> 8;
      const u32x4 ka = {w & 0x000f000fu, w & 0x00f000f0u, w8 & 0x000f000fu, w8 & 0x00f000f0u};
      acc = mfma16x16x32(F16{}, ka, q.op[j], acc);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = __builtin_fmaf(lo_f32(F16{}, c.kp[i].w[g]), acc[i], s[i]);
  }
}

// Online softmax of a tile's scores: weights p (the running maximum moves
// lazily, as in compute_tile).
template <int D>
__device__ __forceinline__ void i4_softmax(const float (&s)[4], float mul, WaveState<D>& st, float (&p)[4]) {
  const float lmax = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])) * mul;
  if (__any(lmax > st.m + kLazyMax)) {
    const float m_new = fmaxf(st.m, wave_max_xor16_32(lmax));
    const float alpha = fast_exp2(st.m - m_new);
    st.m = m_new;
    st.l *= alpha;
#pragma unroll
    for (int e = 0; e < D / 16; ++e) st.acc[e] *= alpha;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = fast_exp2(__builtin_fmaf(s[i], mul, -st.m));
  st.l += (p[0] + p[1]) + (p[2] + p[3]);
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

// O^T += V^T P^T.  d-tile e takes code e of every lane's share, for tokens
// (4 grp, 4 grp + 1) and (4 grp + 2, 4 grp + 3).
template <int D, class KV>
__device__ __forceinline__ void i4_pv(const I4Tile<D, KV>& c, const I4Const& ic, const float (&p)[4],
                                      WaveState<D>& st) {
  using C = I4Tile<D, KV>;
  const u32x2 pop = {pack2(F16{}, p[0], p[1]), pack2(F16{}, p[2], p[3])};
#pragma unroll
  for (int h = 0; h < D / 64; ++h) {        // 4 codes of each token
    const int gv = C::NV == 2 ? h >> 1 : 0;
    uint32_t x[2], x8[2];
    f16x2 s[2], m[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      x[t] = gather16(c.v[2 * t].w[h >> 1], c.v[2 * t + 1].w[h >> 1], h & 1);
      x8[t] = x[t] >> 8;
      s[t] = __builtin_bit_cast(f16x2, gather16(c.vp[2 * t].w[gv], c.vp[2 * t + 1].w[gv], 0));
      m[t] = __builtin_bit_cast(f16x2, gather16(c.vp[2 * t].w[gv], c.vp[2 * t + 1].w[gv], 1));
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      u32x2 va;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint32_t w = e & 2 ? x8[t] : x[t];
        const _Float16 b = e & 1 ? (_Float16)-64.0f : (_Float16)-1024.0f;
        const uint32_t biased = e & 1 ? ((w & ic.hi) | ic.bhi) : ((w & ic.lo) | ic.blo);
        const f16x2 n = __builtin_bit_cast(f16x2, biased) + f16x2{b, b};
        va[t] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(n, s[t], m[t]));
      }
      st.acc[4 * h + e] = mfma16x16x16(F16{}, va, pop, st.acc[4 * h + e]);
    }
  }
}

}  // namespace sia
