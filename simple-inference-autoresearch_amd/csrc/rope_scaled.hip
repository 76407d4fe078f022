// Rotary positions from frequencies, of a part of each head, for gfx950.
//
// Pair i of a token at position n is turned by the angle n f_i (frequency f_i per position) and stretched by a factor.
// A table of cosines costs its reads and a row per position that a long context reaches, and one built in fp32 is off by
// n 2^-24 radians, 0.06 at a million.  Here the angle is taken modulo one turn in 64-bit integers: F = frac(f / 2 pi) 2^64
// (f / 2 pi in fp64), and n F mod 2^64 is the fraction of a turn whatever n is; its top 32 bits give a quadrant and a rest
// of at most an eighth of a turn, where the Taylor series of sine and cosine to the 9th and 10th power are off by less
// than 2^-28.  (What remains is F's own error, 2^-52 of the number of turns.)
//
// Memory-bound: q and k once in, once out.  A work-group takes a few tokens: it computes each token's R / 2 pairs of sine
// and cosine once, into LDS, while its first elements are in flight, and every head's items read them there.  An item is
// PP pairs of a head (8: two 16-byte accesses of 16-bit elements), or 2 PP of the elements behind the rotated part.
#include <string.h>

#include <algorithm>

#include "host_util.hpp"
#include "sia_common.hpp"

namespace sia {

struct RopeScaledArgs {
  const char* x[2]; int64_t sb[2], st[2], sh[2];       // q and k, byte strides
  char* o[2]; int64_t ob[2], ot[2], oh[2];
  const char* pos; int64_t p_sb, p_st;                 // element strides
  const char* freq;
  int32_t rows, T, Hq, H, D, R;                        // rows = B T, H = Hq + Hkv
  int32_t tokens;                                      // per work-group
  int32_t pos64, freq64;
  float scale;
  FastDiv dT, dHead, dItems;                           // by T, items of a head, items of a token
  int32_t head_items;                                  // items of a head
  int32_t rot_items;                                   // of them in the rotated part
};

// sine and cosine of `turn` / 2^64 of a turn
__device__ __forceinline__ float2 sincos_turn(uint64_t turn) {
  const uint32_t t = (uint32_t)(turn >> 32);
  const uint32_t quad = (t + 0x20000000u) >> 30;
  const float a = (float)(int32_t)(t - (quad << 30)) * 1.4629180792671596e-9f;   // 2 pi / 2^32
  const float b = a * a;
  float s = __builtin_fmaf(b, 2.7557319e-6f, -1.9841270e-4f);
  s = __builtin_fmaf(b, s, 8.3333333e-3f);
  s = __builtin_fmaf(b, s, -1.6666667e-1f);
  s = __builtin_fmaf(a * b, s, a);
  float c = __builtin_fmaf(b, -2.7557319e-7f, 2.4801587e-5f);
  c = __builtin_fmaf(b, c, -1.3888889e-3f);
  c = __builtin_fmaf(b, c, 4.1666667e-2f);
  c = __builtin_fmaf(b, c, -0.5f);
  c = __builtin_fmaf(b, c, 1.0f);
  const bool swap = (quad & 1u) != 0u;
  const float ys = swap ? c : s, yc = swap ? s : c;
  return float2{(quad & 2u) != 0u ? -ys : ys, ((quad + 1u) & 2u) != 0u ? -yc : yc};
}

template <int BYTES>
struct Words { uint32_t w[BYTES >= 4 ? BYTES / 4 : 1]; };
template <int BYTES>
__device__ __forceinline__ Words<BYTES> get(const char* p) {
  Words<BYTES> r;
  if constexpr (BYTES % 16 == 0) {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const u32x4 x = __builtin_nontemporal_load((const u32x4*)(p + 16 * i));
#pragma unroll
      for (int e = 0; e < 4; ++e) r.w[4 * i + e] = x[e];
    }
  } else if constexpr (BYTES == 8) {
    const u32x2 x = __builtin_nontemporal_load((const u32x2*)p);
    r.w[0] = x[0]; r.w[1] = x[1];
  } else if constexpr (BYTES == 4) {
    r.w[0] = __builtin_nontemporal_load((const uint32_t*)p);
  } else {
    r.w[0] = __builtin_nontemporal_load((const uint16_t*)p);
  }
  return r;
}
template <int BYTES>
__device__ __forceinline__ void put(char* p, const Words<BYTES>& r) {
  if constexpr (BYTES % 16 == 0) {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i)
      __builtin_nontemporal_store(u32x4{r.w[4 * i], r.w[4 * i + 1], r.w[4 * i + 2], r.w[4 * i + 3]}, (u32x4*)(p + 16 * i));
  } else if constexpr (BYTES == 8) {
    __builtin_nontemporal_store(u32x2{r.w[0], r.w[1]}, (u32x2*)p);
  } else if constexpr (BYTES == 4) {
    __builtin_nontemporal_store(r.w[0], (uint32_t*)p);
  } else {
    __builtin_nontemporal_store((uint16_t)r.w[0], (uint16_t*)p);
  }
}
// element i of the words of elements of type T, and all of them back
template <class T, int BYTES>
__device__ __forceinline__ float elem(const Words<BYTES>& r, int i) {
  if constexpr (std::is_same<T, F32>::value) return __builtin_bit_cast(float, r.w[i]);
  else return (i & 1) ? hi_f32(T{}, r.w[i >> 1]) : lo_f32(T{}, r.w[i >> 1]);
}
template <class T, int N>
__device__ __forceinline__ Words<N * T::bytes> words(const float* x) {
  Words<N * T::bytes> r;
  if constexpr (std::is_same<T, F32>::value) {
#pragma unroll
    for (int i = 0; i < N; ++i) r.w[i] = __builtin_bit_cast(uint32_t, x[i]);
  } else if constexpr (N == 1) {
    r.w[0] = pack2(T{}, x[0], 0.f) & 0xffffu;
  } else {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) r.w[i] = pack2(T{}, x[2 * i], x[2 * i + 1]);
  }
  return r;
}

constexpr int kRopeThreads = 256;
constexpr int kRopeMaxSc = 2048;      // (sine, cosine) pairs that a work-group's LDS holds: 16 KB

template <class T, bool IL, int PP>
__global__ __launch_bounds__(kRopeThreads) void rope_scaled_kernel(const RopeScaledArgs a) {
  __shared__ float2 sc[kRopeMaxSc];
  constexpr int ES = T::bytes, N = PP * ES;
  const int row0 = blockIdx.x * a.tokens, nrow = min(a.tokens, a.rows - row0), half = a.R / 2;
  const int token_items = a.H * a.head_items;
  const int items = nrow * token_items;
  // item it -> its two runs of PP elements in and out, and its first pair (-1: copied)
  struct Item { const char* src; char* dst; int gap, pair; };
  auto item = [&](int it) {
    Item r;
    const int t = fdiv(it, a.dItems), i = it - t * token_items;
    const int h = fdiv(i, a.dHead), c = i - h * a.head_items;
    const int row = row0 + t, b = fdiv(row, a.dT), tt = row - b * a.T;
    const int w = h < a.Hq ? 0 : 1, hh = h - (w ? a.Hq : 0);
    r.src = a.x[w] + b * a.sb[w] + tt * a.st[w] + hh * a.sh[w];
    r.dst = a.o[w] + b * a.ob[w] + tt * a.ot[w] + hh * a.oh[w];
    const bool rot = c < a.rot_items;
    const int at = rot ? (IL ? 2 * PP * c : PP * c) : a.R + 2 * PP * (c - a.rot_items);
    r.gap = (rot && !IL ? half : PP) * ES;
    r.pair = rot ? t * half + PP * c : -1;
    r.src += at * ES;
    r.dst += at * ES;
    return r;
  };
  // the first item's elements fly while the sines are computed
  int it = threadIdx.x;
  Item cur{};
  Words<N> wa{}, wb{};
  if (it < items) {
    cur = item(it);
    wa = get<N>(cur.src);
    wb = get<N>(cur.src + cur.gap);
  }
  for (int i = threadIdx.x; i < nrow * half; i += kRopeThreads) {
    const int t = i / half, pair = i - t * half;
    const int row = row0 + t, b = fdiv(row, a.dT), tt = row - b * a.T;
    const int64_t pi = b * a.p_sb + tt * a.p_st;
    const int64_t n = a.pos64 ? ((const int64_t*)a.pos)[pi] : (int64_t)((const int32_t*)a.pos)[pi];
    double f = (a.freq64 ? ((const double*)a.freq)[pair] : (double)((const float*)a.freq)[pair]) * 0.15915494309189535;
    f -= floor(f);
    float2 y = sincos_turn((uint64_t)n * (uint64_t)(f * 18446744073709551616.0));
    y.x *= a.scale;
    y.y *= a.scale;
    sc[i] = y;
  }
  __syncthreads();
  while (it < items) {
    const int next = it + kRopeThreads;
    Item nx{};
    Words<N> na{}, nb{};
    if (next < items) {
      nx = item(next);
      na = get<N>(nx.src);
      nb = get<N>(nx.src + nx.gap);
    }
    if (cur.pair >= 0) {
      float xa[PP], xb[PP];
#pragma unroll
      for (int i = 0; i < PP; ++i) {
        const float2 y = sc[cur.pair + i];
        const float p = IL ? (2 * i < PP ? elem<T>(wa, 2 * i) : elem<T>(wb, PP > 1 ? 2 * i - PP : 0)) : elem<T>(wa, i);
        const float q = IL ? (2 * i + 1 < PP ? elem<T>(wa, 2 * i + 1) : elem<T>(wb, PP > 1 ? 2 * i + 1 - PP : 0))
                           : elem<T>(wb, i);
        float u, v;
        rope_rotate(p, q, y.y, y.x, u, v);
        if constexpr (IL) {
          if (2 * i < PP) xa[2 * i] = u; else xb[PP > 1 ? 2 * i - PP : 0] = u;
          if (2 * i + 1 < PP) xa[2 * i + 1] = v; else xb[PP > 1 ? 2 * i + 1 - PP : 0] = v;
        } else {
          xa[i] = u;
          xb[i] = v;
        }
      }
      wa = words<T, PP>(xa);
      wb = words<T, PP>(xb);
    }
    put<N>(cur.dst, wa);
    put<N>(cur.dst + cur.gap, wb);
    it = next;
    cur = nx;
    wa = na;
    wb = nb;
  }
}

namespace {

template <class T, bool IL>
int launch_rope_scaled_pp(const RopeScaledArgs& a, int pp, dim3 grid, hipStream_t st) {
  if (pp == 8) hipLaunchKernelGGL((rope_scaled_kernel<T, IL, 8>), grid, dim3(kRopeThreads), 0, st, a);
  else if (pp == 4) hipLaunchKernelGGL((rope_scaled_kernel<T, IL, 4>), grid, dim3(kRopeThreads), 0, st, a);
  else hipLaunchKernelGGL((rope_scaled_kernel<T, IL, 1>), grid, dim3(kRopeThreads), 0, st, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? SIA_OK : fail(SIA_ERR_LAUNCH, "rope launch: %s", hipGetErrorString(e));
}
template <class T>
int launch_rope_scaled_t(const RopeScaledArgs& a, bool il, int pp, dim3 grid, hipStream_t st) {
  return il ? launch_rope_scaled_pp<T, true>(a, pp, grid, st) : launch_rope_scaled_pp<T, false>(a, pp, grid, st);
}

bool empty(const sia_tensor* t) {
  for (int d = 0; d < t->ndim; ++d)
    if (t->shape[d] == 0) return true;
  return false;
}

}  // namespace
}  // namespace sia

using namespace sia;

extern "C" int sia_rope_scaled(const sia_tensor* q, const sia_tensor* k, const sia_tensor* positions,
                               const sia_tensor* inv_freq, int32_t rotary_dim, int32_t interleaved, float scale,
                               const sia_tensor* q_out, const sia_tensor* k_out, void* stream) {
  if (q == nullptr || positions == nullptr || inv_freq == nullptr || q_out == nullptr || (k != nullptr) != (k_out != nullptr))
    return fail(SIA_ERR_INVALID_ARGUMENT, "q, positions, inv_freq and q_out are required, and k_out exactly with k");
  const sia_tensor* in[2] = {q, k};
  const sia_tensor* out[2] = {q_out, k_out};
  if (q->ndim != 4) return fail(SIA_ERR_INVALID_ARGUMENT, "q must be (B, T, H, D)");
  const int64_t B = q->shape[0], T = q->shape[1], D = q->shape[3], R = rotary_dim;
  if (q->dtype != SIA_F16 && q->dtype != SIA_BF16 && q->dtype != SIA_F32)
    return fail(SIA_ERR_UNSUPPORTED, "q dtype %s: expected float16, bfloat16 or float32", dtype_name(q->dtype));
  const int es = elem_size(q->dtype);
  RopeScaledArgs a;
  memset(&a, 0, sizeof(a));
  int64_t H = 0;
  for (int w = 0; w < (k != nullptr ? 2 : 1); ++w) {
    const sia_tensor *x = in[w], *o = out[w];
    const char* name = w ? "k" : "q";
    if (x->ndim != 4 || o->ndim != 4) return fail(SIA_ERR_INVALID_ARGUMENT, "%s and its output must be (B, T, H, D)", name);
    if (x->dtype != q->dtype || o->dtype != q->dtype) return fail(SIA_ERR_INVALID_ARGUMENT, "q, k and the outputs must share one dtype");
    if (x->shape[0] != B || x->shape[1] != T || x->shape[3] != D)
      return fail(SIA_ERR_INVALID_ARGUMENT, "k must be (B, T, Hkv, D) with q's B, T and D");
    for (int d = 0; d < 4; ++d)
      if (o->shape[d] != x->shape[d]) return fail(SIA_ERR_INVALID_ARGUMENT, "output shape differs from its input");
    if ((x->stride[3] != 1 || o->stride[3] != 1) && D > 1)
      return fail(SIA_ERR_INVALID_ARGUMENT, "%s and its output must be contiguous along head_dim", name);
    if (!empty(x) && (x->data == nullptr || o->data == nullptr))
      return fail(SIA_ERR_INVALID_ARGUMENT, "a non-empty tensor has no data pointer");
    H += x->shape[2];
    a.x[w] = (const char*)x->data; a.sb[w] = bstride(x, 0); a.st[w] = bstride(x, 1); a.sh[w] = bstride(x, 2);
    a.o[w] = (char*)o->data; a.ob[w] = bstride(o, 0); a.ot[w] = bstride(o, 1); a.oh[w] = bstride(o, 2);
  }
  if (R < 2 || R % 2 || R > D) return fail(SIA_ERR_INVALID_ARGUMENT, "rotary_dim %d must be even, at least 2 and at most head_dim %lld", rotary_dim, (long long)D);
  if (R / 2 > kRopeMaxSc) return fail(SIA_ERR_UNSUPPORTED, "rotary_dim %d exceeds %d", rotary_dim, 2 * kRopeMaxSc);
  if (positions->dtype != SIA_I32 && positions->dtype != SIA_I64)
    return fail(SIA_ERR_INVALID_ARGUMENT, "positions must be int32 or int64");
  if (!((positions->ndim == 1 && positions->shape[0] == T) ||
        (positions->ndim == 2 && positions->shape[0] == B && positions->shape[1] == T)))
    return fail(SIA_ERR_INVALID_ARGUMENT, "positions must be (T,) or (B, T)");
  if ((inv_freq->dtype != SIA_F32 && inv_freq->dtype != SIA_F64) || inv_freq->ndim != 1 || inv_freq->shape[0] != R / 2 ||
      inv_freq->data == nullptr || (R > 2 && inv_freq->stride[0] != 1))
    return fail(SIA_ERR_INVALID_ARGUMENT, "inv_freq must be a contiguous float32 or float64 (rotary_dim / 2,) tensor");
  if (B * T == 0 || H == 0) return SIA_OK;
  if (positions->data == nullptr) return fail(SIA_ERR_INVALID_ARGUMENT, "positions has no data pointer");
  if (B * T > 0x7fffffff || H * D > 0x7fffff) return fail(SIA_ERR_UNSUPPORTED, "too many rows or heads");
  a.pos = (const char*)positions->data;
  a.p_sb = positions->ndim == 2 ? positions->stride[0] : 0;
  a.p_st = positions->stride[positions->ndim - 1];
  a.pos64 = positions->dtype == SIA_I64;
  a.freq = (const char*)inv_freq->data;
  a.freq64 = inv_freq->dtype == SIA_F64;
  a.rows = (int32_t)(B * T); a.T = (int32_t)T; a.Hq = (int32_t)q->shape[2]; a.H = (int32_t)H;
  a.D = (int32_t)D; a.R = (int32_t)R;
  a.scale = scale;
  // the widest items whose runs of elements start at multiples of their size (at most 16 bytes) everywhere
  int pp = 1;
  for (const int p : {8, 4}) {
    const int64_t al = std::min(16, p * es);
    bool ok = (R / 2) % p == 0 && (D - R) % (2 * p) == 0;
    for (int w = 0; w < (k != nullptr ? 2 : 1); ++w) {
      const int64_t at[] = {(int64_t)(uintptr_t)a.x[w], (int64_t)(uintptr_t)a.o[w], a.sb[w], a.st[w], a.sh[w], a.ob[w], a.ot[w], a.oh[w]};
      for (const int64_t x : at) ok = ok && x % al == 0;
    }
    if (ok) {
      pp = p;
      break;
    }
  }
  a.rot_items = (int32_t)(R / 2 / pp);
  // (single elements: what lies behind the rotated part is an even number of them, as D and R are, or D is refused)
  if ((D - R) % (2 * pp) != 0) return fail(SIA_ERR_UNSUPPORTED, "head_dim %lld must be even", (long long)D);
  a.head_items = a.rot_items + (int32_t)((D - R) / (2 * pp));
  a.dT = make_fastdiv((uint32_t)T);
  a.dHead = make_fastdiv((uint32_t)a.head_items);
  a.dItems = make_fastdiv((uint32_t)(H * a.head_items));
  int rc;
  if ((rc = device_ok())) return rc;
  // tokens per work-group: as many as leave four groups per CU, at most 4 items a thread and the sines that fit
  int64_t tokens = std::max<int64_t>(1, 4LL * kRopeThreads / (H * a.head_items));
  tokens = std::min(tokens, std::max<int64_t>(1, (B * T) / (4LL * device_info().cus)));
  tokens = std::min<int64_t>(tokens, kRopeMaxSc / (R / 2));
  a.tokens = (int32_t)tokens;
  const dim3 grid((unsigned)((B * T + tokens - 1) / tokens));
  const hipStream_t st = (hipStream_t)stream;
  switch (q->dtype) {
    case SIA_F16: return launch_rope_scaled_t<F16>(a, interleaved != 0, pp, grid, st);
    case SIA_BF16: return launch_rope_scaled_t<BF16>(a, interleaved != 0, pp, grid, st);
    default: return launch_rope_scaled_t<F32>(a, interleaved != 0, pp, grid, st);
  }
}
