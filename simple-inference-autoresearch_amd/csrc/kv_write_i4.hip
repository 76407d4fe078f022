// KV writes into 4-bit destinations (the format: int4.hpp), with RoPE of K and
// q on the way when asked for, like kv_write.hip.
//
// A lane owns the words of a row that stand together in 16 bytes of codes
// (32 elements; 64 at head_dim 256, whose two blocks it takes both), so 4 lanes
// make a row of 128 elements or more, 2 one of 64, 1 a shorter one:
//  * a group of 32 is then one word of each of the four lanes (2 words of two, 4
//    of one), and its extremes take two exchanges inside a quad of lanes;
//  * the codes leave in one 16-byte store;
//  * the elements of a split-half rotary pair are in one lane.
//
// Bound: HBM, with the vector ALU close behind.  Per element: x - m, the quotient
// (div_by_scale), a clamp, a rounding by adding 1.5 2^23, one shift-and-add into
// the word; 11 instructions with the extremes.  4 x 8192 tokens, 16 heads of 64,
// fp16, groups of 64: 40.2 us, 172 MB at 4.3 TB/s.  (A lane per 8 elements, with
// rounding, conversion and packing on their own and 64-bit addresses for every
// word, took 36 instructions and 62.9 us.)
//
// Rows are ordered so that 16 tokens of one head are neighbours: a work-group
// completes the lines that it stores (16 tokens' parameters are 64 to 256
// bytes), where lines shared between work-groups, and so between L2s, are
// written to memory in parts.
#include "host_util.hpp"
#include "int4.hpp"
#include "kv_rows.hpp"
#include "kv_write.hpp"

namespace sia {

template <int D>
struct I4Row {
  static constexpr int LR = D >= 128 ? 4 : D == 64 ? 2 : 1;   // lanes of a row
  static constexpr int WL = D / 8 / LR;                       // words of a lane
  // Word j of lane q: the words at places [4 q, 4 q + 4) of a block.
  static __device__ __forceinline__ int word(int q, int j) {
    if constexpr (D >= 128) return q + 4 * j;
    else if constexpr (D == 64) return 2 * q + (j & 1) * 4 + (j >> 1);
    else return j;
  }
  // The word of the same lane that holds word j's split-half partners.
  static constexpr int partner(int j) { return D >= 128 ? j + WL / 2 : D == 64 ? j ^ 1 : j + WL / 2; }
  static constexpr bool first_half(int j) { return D == 64 ? (j & 1) == 0 : j < WL / 2; }
};

// Largest and smallest with NaN winning.
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float min_nan(float a, float b) { return __builtin_elementwise_minimum(a, b); }

template <int CTRL>
__device__ __forceinline__ float quad(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, false));
}

// Parameters of a group with extremes lo and hi (NaN if any element is): s low, m high.
// *s, *inv: the step and its reciprocal (0 for a step of 0); *m the minimum.
__device__ __forceinline__ uint32_t i4_group_params(float lo, float hi, float* s, float* inv, float* m, bool* poison) {
#pragma clang fp contract(off)
  *poison = !(hi <= 3.402823466e38f && lo >= -3.402823466e38f);
  lo = __builtin_amdgcn_fmed3f(lo, -kF16Max, kF16Max);
  hi = __builtin_amdgcn_fmed3f(hi, -kF16Max, kF16Max);
  const _Float16 mh = (_Float16)lo;
  *m = (float)mh;
  // (hi - m) / 15 correctly rounded (div_by_scale's correction step)
  const float step = fmaxf(div_by_scale(hi - *m, 15.0f, 1.0f / 15.0f), 0.0f);
  const uint32_t sbits = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(step, 0.0f)) & 0xffffu;
  *s = lo_f32(F16{}, sbits);
  // 1 / s: v_rcp_f32 is within an ulp, and one Newton step under FMAs rounds
  // it correctly for every fp16 s (tests/test_int4_format.py)
  const float r = __builtin_amdgcn_rcpf(*s);
  *inv = *s > 0.0f ? __builtin_fmaf(__builtin_fmaf(-*s, r, 1.0f), r, r) : 0.0f;
  return *poison ? 0x7e007e00u : sbits | ((uint32_t)__builtin_bit_cast(uint16_t, mh) << 16);
}

// 8 elements as a word of codes.
__device__ __forceinline__ uint32_t i4_word_of(const float* x, float s, float inv, float m, bool clamp) {
#pragma clang fp contract(off)
  // adding 1.5 2^23 leaves the value rounded (half to even) in the low bits of
  // the sum; what its exponent adds to the word is the same for every word
  constexpr float kMagic = 12582912.0f;
  constexpr uint32_t kBits = 0x4b400000u;
  uint32_t w = 0u - (kBits + (kBits << 4) + (kBits << 8) + (kBits << 12) + (kBits << 16) + (kBits << 20) +
                     (kBits << 24) + (kBits << 28));
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float v = clamp ? __builtin_amdgcn_fmed3f(x[i], -kF16Max, kF16Max) : x[i];
    const float n = __builtin_amdgcn_fmed3f(div_by_scale(v - m, s, inv), 0.0f, 15.0f);
    w += __builtin_bit_cast(uint32_t, n + kMagic) << (4 * i);
  }
  return w;
}

// Table values of 8 consecutive columns from j0 of a row, whatever the table's dtype (uniform).
__device__ __forceinline__ void tab8(const KvWriteArgs& a, const char* row, int j0, float* c) {
  if (a.tab_dt == SIA_F32) tab_n<F32, 8>(row, j0, c);
  else if (a.tab_dt == SIA_F16) tab_n<F16, 8>(row, j0, c);
  else tab_n<BF16, 8>(row, j0, c);
}

typedef uint32_t u32x2_a4 __attribute__((ext_vector_type(2), aligned(4)));
typedef uint32_t u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

template <class S, int D, int ROPE>
__global__ __launch_bounds__(256) void kv_write_i4(const KvWriteArgs a) {
  using R = I4Row<D>;
  constexpr int LR = R::LR, WL = R::WL;
  if constexpr (ROPE != 0) {
    if (blockIdx.x >= a.kv_blocks) {                            // whole work-group in the q part
      if (blockIdx.y != 0) return;
      const uint32_t token = blockIdx.x - a.kv_blocks;
      if (a.tab_dt == SIA_F32) rope_q_token<S, F32, ROPE>(a, token);
      else if (a.tab_dt == SIA_F16) rope_q_token<S, F16, ROPE>(a, token);
      else rope_q_token<S, BF16, ROPE>(a, token);
      return;
    }
  }
  const int which = blockIdx.y;                                 // 0: K, 1: V
  const uint32_t gid = blockIdx.x * 256u + threadIdx.x;         // (the host keeps rows * LR below 2^31)
  const int q = (int)(gid % LR);
  const uint32_t row_raw = gid / LR;
  const bool live_row = row_raw < (uint32_t)a.rows;
  const uint32_t row = live_row ? row_raw : (uint32_t)a.rows - 1u;
  const int rest = (int)(row >> a.lg_chunk);
  const int bc = fdiv(rest, a.dH), h = rest - bc * a.H;
  const int b = fdiv(bc, a.dchunks);
  const int chunks = (a.T + (1 << a.lg_chunk) - 1) >> a.lg_chunk;
  int t = ((bc - b * chunks) << a.lg_chunk) + (int)(row & ((1u << a.lg_chunk) - 1u));
  const bool live_token = live_row && t < a.T;
  t = min(t, a.T - 1);
  const int64_t pos = (int64_t)t + a.start_host + (a.start ? a.start[a.start_per_seq ? b : 0] : 0);
  const bool in_range = live_token && pos >= 0 && pos < a.cap && (ROPE == 0 || pos < a.Tc);
  const int pos_c = in_range ? (int)pos : 0;
  const char* src = (which ? a.src1 : a.src0) + ((int64_t)b * a.s_sb + (int64_t)h * a.s_sh + (int64_t)t * a.s_st);
  float x[WL][8];
#pragma unroll
  for (int j = 0; j < WL; ++j) load8<S>(src + R::word(q, j) * 8 * S::bytes, x[j]);
  // destination slot (page-table entry 0 of the row's sequence when out of range)
  int64_t slot0 = b, slot1 = pos_c;
  bool ok = in_range;
  if (a.paged) {
    const int blk = fdiv(pos_c, a.dpage);
    const int pg = a.bt[(int64_t)b * a.bt_sb + (int64_t)blk * a.bt_sl];
    ok = ok && pg >= 0 && (int64_t)pg < a.num_pages;
    slot0 = pg;
    slot1 = pos_c - blk * a.page;
  }
  if constexpr (ROPE != 0) {
    if (which == 0) {                                           // (uniform) K, rounded to its dtype afterwards
      const char* crow = a.cs + (int64_t)pos_c * a.tab_rs;
      const char* srow = a.sn + (int64_t)pos_c * a.tab_rs;
#pragma unroll
      for (int j = 0; j < WL; ++j) {
        float c[8], s[8];
        const int e0 = 8 * R::word(q, j);
        if constexpr (ROPE == 1) {
          if (!R::first_half(j)) continue;
          tab8(a, crow, e0, c);
          tab8(a, srow, e0, s);
          float* y = x[R::partner(j)];
#pragma unroll
          for (int i = 0; i < 8; ++i) rope_rotate(x[j][i], y[i], c[i], s[i], x[j][i], y[i]);
        } else {
          // (4 pairs: table columns e0 / 2 .. e0 / 2 + 3, inside one aligned 8)
          tab8(a, crow, (e0 / 2) & ~7, c);
          tab8(a, srow, (e0 / 2) & ~7, s);
          const bool up = (e0 / 2) & 4;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            rope_rotate(x[j][2 * k], x[j][2 * k + 1], up ? c[4 + k] : c[k], up ? s[4 + k] : s[k], x[j][2 * k],
                        x[j][2 * k + 1]);
        }
      }
#pragma unroll
      for (int j = 0; j < WL; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[j][i] = to_src<S>(x[j][i]);
    }
  }
  // extremes of the units of min(D, 32) elements: all lanes of the row (D >=
  // 128: one word each; 64: two) or one lane
  constexpr int NU = D / 32 > 0 ? D / 32 : 1;
  float lo[NU], hi[NU];
#pragma unroll
  for (int u = 0; u < NU; ++u) {
    bool first = true;
#pragma unroll
    for (int j = 0; j < WL; ++j) {
      // unit of word j, the same for every lane: word / 4
      const int uj = D >= 128 ? j : D == 64 ? (j & 1) : 0;
      if (uj != u) continue;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        lo[u] = first ? x[j][i] : min_nan(lo[u], x[j][i]);
        hi[u] = first ? x[j][i] : max_nan(hi[u], x[j][i]);
        first = false;
      }
    }
    if constexpr (LR >= 2) {
      lo[u] = min_nan(lo[u], quad<0xb1>(lo[u]));              // lane ^ 1
      hi[u] = max_nan(hi[u], quad<0xb1>(hi[u]));
    }
    if constexpr (LR >= 4) {
      lo[u] = min_nan(lo[u], quad<0x4e>(lo[u]));              // lane ^ 2
      hi[u] = max_nan(hi[u], quad<0x4e>(hi[u]));
    }
  }
  // units of one group (uniform: 1, 2 or 4)
  if (D >= 64 && a.lg_group >= 6) {
#pragma unroll
    for (int u = 0; u < NU; u += 2)
      if (u + 1 < NU) {
        lo[u] = lo[u + 1] = min_nan(lo[u], lo[u + 1]);
        hi[u] = hi[u + 1] = max_nan(hi[u], hi[u + 1]);
      }
  }
  if (D >= 128 && a.lg_group >= 7) {
#pragma unroll
    for (int u = 0; u + 2 < NU; u += 4) {
      const float l = min_nan(lo[u], lo[u + 2]), g = max_nan(hi[u], hi[u + 2]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        lo[u + k] = l;
        hi[u + k] = g;
      }
    }
  }
  uint32_t sm[NU], w[WL];
#pragma unroll
  for (int u = 0; u < NU; ++u) {
    float s, inv, m;
    bool poison;
    sm[u] = i4_group_params(lo[u], hi[u], &s, &inv, &m, &poison);
#pragma unroll
    for (int j = 0; j < WL; ++j) {
      const int uj = D >= 128 ? j : D == 64 ? (j & 1) : 0;
      if (uj != u) continue;
      w[j] = poison ? 0u : i4_word_of(x[j], s, inv, m, !std::is_same<S, F16>::value);
    }
  }
  if (!ok) return;
  char* dst = (which ? a.dst1 : a.dst0) + (slot0 * a.d_s0 + (int64_t)h * a.d_sh + slot1 * a.d_sn);
  char* par = (which ? a.sc1 : a.sc0) + (slot0 * a.c_s0 + (int64_t)h * a.c_sh + slot1 * a.c_sn);
  // (8-byte aligned rows)
  if constexpr (D == 16) {
    *(u32x2*)dst = u32x2{w[0], w[1]};
  } else {
#pragma unroll
    for (int k = 0; k < WL / 4; ++k)
      *(u32x4_a4*)(dst + 64 * k + 16 * q) = u32x4_a4{w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]};
  }
  if (q != 0) return;
  if constexpr (NU == 1) {
    *(uint32_t*)par = sm[0];
  } else if (a.lg_group == 5) {
    if constexpr (NU == 2) *(u32x2_a4*)par = u32x2_a4{sm[0], sm[1]};
    else
#pragma unroll
      for (int u = 0; u < NU; u += 4) *(u32x4_a4*)(par + 4 * u) = u32x4_a4{sm[u], sm[u + 1], sm[u + 2], sm[u + 3]};
  } else if (a.lg_group == 6) {
    if constexpr (NU == 2) *(uint32_t*)par = sm[0];
    else if constexpr (NU == 4) *(u32x2_a4*)par = u32x2_a4{sm[0], sm[2]};
    else *(u32x4_a4*)par = u32x4_a4{sm[0], sm[2], sm[4 % NU], sm[6 % NU]};
  } else {
    if constexpr (NU == 8) *(u32x2_a4*)par = u32x2_a4{sm[0], sm[4 % NU]};
    else *(uint32_t*)par = sm[0];
  }
}

template <class S, int D>
static int launch_i4_rope(const KvWriteArgs& a, hipStream_t stream) {
  const int64_t q_blocks = a.rope != 0 && a.q && a.Hq > 0 ? (int64_t)a.B * a.T : 0;   // one per token
  if (a.kv_blocks + q_blocks > 0x7fffffff) return fail(SIA_ERR_UNSUPPORTED, "too many rows for one launch");
  const dim3 grid((unsigned)(a.kv_blocks + q_blocks), (unsigned)a.ntensors);
  switch (a.rope) {
    case 1: hipLaunchKernelGGL((kv_write_i4<S, D, 1>), grid, dim3(256), 0, stream, a); break;
    case 2: hipLaunchKernelGGL((kv_write_i4<S, D, 2>), grid, dim3(256), 0, stream, a); break;
    default: hipLaunchKernelGGL((kv_write_i4<S, D, 0>), grid, dim3(256), 0, stream, a); break;
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(SIA_ERR_LAUNCH, "kv write launch: %s", hipGetErrorString(e));
  return SIA_OK;
}

template <class S>
static int launch_i4_d(const KvWriteArgs& a, hipStream_t stream) {
  switch (a.D) {
    case 16: return launch_i4_rope<S, 16>(a, stream);
    case 32: return launch_i4_rope<S, 32>(a, stream);
    case 64: return launch_i4_rope<S, 64>(a, stream);
    case 128: return launch_i4_rope<S, 128>(a, stream);
    case 256: return launch_i4_rope<S, 256>(a, stream);
    default: return fail(SIA_ERR_UNSUPPORTED, "head_dim %d not supported", a.D);
  }
}

int launch_kv_write_i4(const KvWriteArgs& a_in, int src_dtype, hipStream_t stream) {
  KvWriteArgs a = a_in;
  const int lanes = a.D >= 128 ? 4 : a.D == 64 ? 2 : 1;
  a.lg_chunk = a.T >= 16 ? 4 : 0;
  const int64_t chunks = (a.T + (1 << a.lg_chunk) - 1) >> a.lg_chunk;
  a.rows = (int64_t)a.B * chunks * a.H << a.lg_chunk;
  if (a.rows * lanes + 255 > 0x7fffffff || (int64_t)a.B * a.T > 0x7fffffff)
    return fail(SIA_ERR_UNSUPPORTED, "too many rows for one launch");
  if (a.rows == 0 && (a.rope == 0 || a.q == nullptr || a.q_rows == 0)) return SIA_OK;
  a.kv_blocks = (uint32_t)((a.rows * lanes + 255) / 256);
  a.dH = make_fastdiv((uint32_t)(a.H > 0 ? a.H : 1));
  a.dchunks = make_fastdiv((uint32_t)(chunks > 0 ? chunks : 1));
  a.paged = a.bt != nullptr && a.cap > 0 ? 1 : 0;
  if (a.paged) a.dpage = make_fastdiv((uint32_t)a.page);
  switch (src_dtype) {
    case SIA_F16: return launch_i4_d<F16>(a, stream);
    case SIA_BF16: return launch_i4_d<BF16>(a, stream);
    case SIA_F32: return launch_i4_d<F32>(a, stream);
    default: return fail(SIA_ERR_UNSUPPORTED, "source dtype %s not supported", dtype_name(src_dtype));
  }
}

}  // namespace sia
