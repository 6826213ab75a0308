// pkv_append.cu — the way into the paged cache: rotary embedding and KV-append
// of any step in one launch, and the page index (int8 key bounds per page and
// KV head) that page-sparse attention scores pages with.
//
//   rope_append_kernel   q' = R(pos) q -> q_out, k' = R(pos) k and v -> their
//                        slots. R turns pair i of each head by the angle whose
//                        cosine / sine are the tables' row `pos`, entry i; the
//                        pair is (i, i + rot/2), or (2i, 2i + 1) interleaved;
//                        dims rot.. of a head pass through. Products are
//                        rounded to fp32 before the difference / sum
//                        (rope_pair), then once to the pool dtype: the bits of
//                        pkv_rope followed by pkv_append_kv.
//   page_index_kernel    bounds of whole pages: lo / hi = elementwise min / max
//                        of the page's keys, scale = max(|lo|, |hi|) / 127,
//                        codes floor(lo / scale), ceil(hi / scale).
//                        A NaN key makes the scale NaN (and the codes 0), so that
//                        its page scores no number, above every number; an
//                        infinite one makes it infinite: +-127 for infinite
//                        bounds, 0 for the others.
//
// Both move each byte once and do a few operations on it: HBM bound. 16384 tokens
// of 32 + 8 + 8 heads of 64 (fp16, 203 MB): 36 us = 5.6 TB/s (0.87 of the copy
// rate); with the index of their 1024 pages, a second launch, 44 us. A step of a
// few tokens is a launch (2.6 us). Indexing inside the append, each completed page
// by the CTA of its last token from the tokens' k rotated again, took 53 to 58 us
// for that step (139 -> 145 registers, or spills at 80): not kept.
#include <algorithm>
#include <type_traits>

#include "pkv_common.cuh"

namespace pkv {
namespace {

struct RopeAppendArgs {
  const char* q;
  const char* k;
  const char* v;
  char* q_out;
  char* k_slab;
  char* v_slab;
  const int32_t* slots;
  const int64_t* positions;
  const float* cs;
  const float* sn;
  int32_t* st;
  int64_t q_stride, k_stride, v_stride, qo_stride;  // bytes between tokens
  int64_t n_tokens, n_slots, max_pos;
  int hq, hkv, d, half;  // half = rotated pairs per head
  int wpt;               // warps per token
  int cols;              // lanes side by side on a head's columns (vectors): a power of two
};

template <typename T>
__device__ __forceinline__ void unpack_vec(const uint4& u, float (&f)[16 / sizeof(T)]) {
  if constexpr (sizeof(T) == 4) {
    f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
  } else {
    const float2 a = unpack2<T>(u.x), b = unpack2<T>(u.y), c = unpack2<T>(u.z), d = unpack2<T>(u.w);
    f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y; f[4] = c.x; f[5] = c.y; f[6] = d.x; f[7] = d.y;
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack_vec(const float (&f)[16 / sizeof(T)]) {
  if constexpr (sizeof(T) == 4)
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  else
    return make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
}

template <typename T>
__device__ __forceinline__ uint32_t min_word(uint32_t a, uint32_t b) {
  if constexpr (sizeof(T) == 4) {
    return __float_as_uint(fmin_nan(__uint_as_float(a), __uint_as_float(b)));
  } else if constexpr (std::is_same<T, __half>::value) {
    const __half2 m = __hmin2_nan(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  } else {
    const __nv_bfloat162 m =
        __hmin2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
}
template <typename T>
__device__ __forceinline__ uint32_t max_word(uint32_t a, uint32_t b) {
  if constexpr (sizeof(T) == 4) {
    return __float_as_uint(fmax_nan(__uint_as_float(a), __uint_as_float(b)));
  } else if constexpr (std::is_same<T, __half>::value) {
    const __half2 m = __hmax2_nan(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  } else {
    const __nv_bfloat162 m =
        __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
}
template <typename T>
__device__ __forceinline__ uint4 min_words(const uint4& a, const uint4& b) {
  return make_uint4(min_word<T>(a.x, b.x), min_word<T>(a.y, b.y), min_word<T>(a.z, b.z), min_word<T>(a.w, b.w));
}
template <typename T>
__device__ __forceinline__ uint4 max_words(const uint4& a, const uint4& b) {
  return make_uint4(max_word<T>(a.x, b.x), max_word<T>(a.y, b.y), max_word<T>(a.z, b.z), max_word<T>(a.w, b.w));
}
__device__ __forceinline__ uint4 shfl_xor4(const uint4& a, int off) {
  return make_uint4(__shfl_xor_sync(0xffffffffu, a.x, off), __shfl_xor_sync(0xffffffffu, a.y, off),
                    __shfl_xor_sync(0xffffffffu, a.z, off), __shfl_xor_sync(0xffffffffu, a.w, off));
}

__device__ __forceinline__ uint32_t word_of(const uint4& v, int w) {
  return w == 0 ? v.x : w == 1 ? v.y : w == 2 ? v.z : v.w;
}
// largest magnitude of a word of bounds
template <typename T>
__device__ __forceinline__ float top_of_word(uint32_t lo, uint32_t hi) {
  if constexpr (sizeof(T) == 4) {
    return fmax_nan(fabsf(__uint_as_float(lo)), fabsf(__uint_as_float(hi)));
  } else {
    const float2 a = unpack2<T>(lo), b = unpack2<T>(hi);
    return fmax_nan(fmax_nan(fabsf(a.x), fabsf(a.y)), fmax_nan(fabsf(b.x), fabsf(b.y)));
  }
}
// An infinite bound (its scale is infinite too: the finite ones' codes are 0) is
// the extreme code of its sign; a scale of 0 or NaN gives 0.
__device__ __forceinline__ int8_t code_of(float x, float scale, bool up) {
  float y = scale > 0.f ? (up ? ceilf(__fdiv_rn(x, scale)) : floorf(__fdiv_rn(x, scale))) : 0.f;
  if (fabsf(x) == INFINITY && scale > 0.f) y = x;
  return int8_t(fminf(fmaxf(y, -127.f), 127.f));
}
// Codes of a word of bounds: floor(lo / scale) at c, ceil(hi / scale) at c + d,
// clamped; 0 where the scale is 0.
template <typename T>
__device__ __forceinline__ void store_codes(int8_t* c, int d, uint32_t lo, uint32_t hi, float scale) {
  if constexpr (sizeof(T) == 4) {
    c[0] = code_of(__uint_as_float(lo), scale, false);
    c[d] = code_of(__uint_as_float(hi), scale, true);
  } else {
    const float2 a = unpack2<T>(lo), b = unpack2<T>(hi);
    *reinterpret_cast<char2*>(c) = make_char2(code_of(a.x, scale, false), code_of(a.y, scale, false));
    *reinterpret_cast<char2*>(c + d) = make_char2(code_of(b.x, scale, true), code_of(b.y, scale, true));
  }
}

template <typename T, int VE, bool INTER>
__device__ __forceinline__ void turn_pair(float (&p)[VE], float (&r)[VE], const float (&c)[VE], const float (&s)[VE]) {
  if constexpr (INTER) {
#pragma unroll
    for (int e = 0; e < VE; e += 2) {
      rope_pair(p[e], p[e + 1], c[e / 2], s[e / 2]);
      rope_pair(r[e], r[e + 1], c[VE / 2 + e / 2], s[VE / 2 + e / 2]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e) rope_pair(p[e], r[e], c[e], s[e]);
  }
}
template <int VE>
__device__ __forceinline__ void load_angles(const float* p, float (&f)[VE]) {
#pragma unroll
  for (int e = 0; e < VE; e += 4) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(p + e));
    f[e] = v.x; f[e + 1] = v.y; f[e + 2] = v.z; f[e + 3] = v.w;
  }
}

// One token's work, shared by wpt warps. VECTOR: 16-byte vectors of VE
// elements; a lane owns one column of VE pairs (its cosines and sines stay in
// registers) and steps over the heads, UB of them loaded before the first is
// stored, so that a token's rows travel together (16384 tokens of 32 + 8 + 8
// heads of 64: UB 5 36 us, 4 39.5, 2 43; at two CTAs per SM). Otherwise single
// elements.
template <typename T, bool VECTOR, bool INTER>
__global__ void __launch_bounds__(256, 2) rope_append_kernel(const RopeAppendArgs a) {
  constexpr int VE = VECTOR ? 16 / int(sizeof(T)) : 1;
  constexpr int UB = 5;
  using V = typename std::conditional<VECTOR, uint4, T>::type;
  pdl_trigger();
  pdl_wait();  // q, k, v, positions and slots may come from the kernels just before
  const int lane = threadIdx.x & 31;
  const int64_t warp = (int64_t(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  const int64_t t = warp / a.wpt;
  if (t >= a.n_tokens) return;
  const int u0 = int(warp - t * a.wpt) * 32 + lane, du = a.wpt * 32;
  const int64_t pos = a.positions[t], slot = a.slots[t];
  const bool turn = pos >= 0 && pos < a.max_pos;
  const bool store = slot >= 0 && slot < a.n_slots;
  const int d = a.d, half = a.half, heads = a.hq + a.hkv;
  const int64_t row = int64_t(a.hkv) * d * sizeof(T);
  const T* q = reinterpret_cast<const T*>(a.q + t * a.q_stride);
  const T* k = reinterpret_cast<const T*>(a.k + t * a.k_stride);
  T* qo = reinterpret_cast<T*>(a.q_out + t * a.qo_stride);
  T* ko = reinterpret_cast<T*>(a.k_slab + (store ? slot * row : 0));
  // the token's v: its first vectors are loaded now and stored last
  const V* vs = reinterpret_cast<const V*>(a.v + t * a.v_stride);
  const int nv = a.hkv * d / VE;
  V vv[UB];
#pragma unroll
  for (int b = 0; b < UB; ++b)
    if (u0 + b * du < nv) vv[b] = vs[u0 + b * du];
  if (u0 == 0) {
    if (!turn) flag(a.st, PKV_DEV_META_BAD);
    if (!store) flag(a.st, PKV_DEV_SLOT_OOB);
  }
  const float* cs = a.cs + (turn ? pos : 0) * half;
  const float* sn = a.sn + (turn ? pos : 0) * half;
  auto src = [&](int hh) -> const T* { return hh < a.hq ? q + hh * d : k + (hh - a.hq) * d; };
  // NULL: a key whose slot is outside the pool
  auto dst = [&](int hh) -> T* { return hh < a.hq ? qo + hh * d : (store ? ko + (hh - a.hq) * d : nullptr); };

  if constexpr (VECTOR) {
    const int cols = half / VE;  // <= a.cols, a power of two <= 32
    const int i = (lane & (a.cols - 1)) * VE, step = du / a.cols;
    // half-split: elements i.. and half + i..; interleaved: the 2 VE elements from 2 i
    const int e0 = INTER ? 2 * i : i, e1 = INTER ? 2 * i + VE : half + i;
    const int h0 = i < cols * VE ? u0 / a.cols : heads;
    float c[VE], s[VE];
    if (h0 < heads) {
      load_angles<VE>(cs + i, c);
      load_angles<VE>(sn + i, s);
    }
    for (int hb = h0; hb < heads; hb += UB * step) {
      uint4 xa[UB], xb[UB];
#pragma unroll
      for (int b = 0; b < UB; ++b)
        if (hb + b * step < heads) {
          const T* x = src(hb + b * step);
          xa[b] = *reinterpret_cast<const uint4*>(x + e0);
          xb[b] = *reinterpret_cast<const uint4*>(x + e1);
        }
#pragma unroll
      for (int b = 0; b < UB; ++b) {
        if (hb + b * step >= heads) continue;
        float p[VE], r[VE];
        unpack_vec<T>(xa[b], p);
        unpack_vec<T>(xb[b], r);
        if (turn) turn_pair<T, VE, INTER>(p, r, c, s);
        if (T* y = dst(hb + b * step)) {
          *reinterpret_cast<uint4*>(y + e0) = pack_vec<T>(p);
          *reinterpret_cast<uint4*>(y + e1) = pack_vec<T>(r);
        }
      }
    }
  } else {
    for (int u = u0; u < heads * half; u += du) {
      const int hh = u / half, i = u - hh * half;
      const int e0 = INTER ? 2 * i : i, e1 = INTER ? 2 * i + 1 : half + i;
      const T* x = src(hh);
      float p = to_f<T>(x[e0]), r = to_f<T>(x[e1]);
      if (turn) rope_pair(p, r, cs[i], sn[i]);
      if (T* y = dst(hh)) {
        y[e0] = from_f<T>(p);
        y[e1] = from_f<T>(r);
      }
    }
  }
  const int pass = (d - 2 * half) / VE;  // pass-through vectors per head
  for (int u = u0; u < heads * pass; u += du) {
    const int hh = u / pass, e = 2 * half + (u - hh * pass) * VE;
    const V w = *reinterpret_cast<const V*>(src(hh) + e);
    if (T* y = dst(hh)) *reinterpret_cast<V*>(y + e) = w;
  }
  if (store) {
    V* vo = reinterpret_cast<V*>(a.v_slab + slot * row);
#pragma unroll
    for (int b = 0; b < UB; ++b)
      if (u0 + b * du < nv) vo[u0 + b * du] = vv[b];
    for (int u = u0 + UB * du; u < nv; u += du) vo[u] = vs[u];
  }
}

// ---------------------------------------------------------------- page index
struct IndexArgs {
  const char* k_base;   // layer 0's K slab
  int8_t* codes;        // [layers][num_blocks][n_kv][2][d]
  float* scales;        // [layers][num_blocks][n_kv]
  const int32_t* ids;   // slots of the step's tokens (layer >= 0) or block ids (layer < 0: every layer)
  int32_t* st;
  int64_t n, num_blocks, slab_bytes;
  int layer, num_layers, hkv, d, page;
};

constexpr int IX_MAX_EPL = 8;  // head_dim <= 256

// One warp: index entry of KV head h of block `blk`, layer `layer`.
template <typename T>
__device__ __forceinline__ void index_entry(const IndexArgs& a, int layer, int64_t blk, int h, int lane) {
  const int d = a.d;
  const T* k = reinterpret_cast<const T*>(a.k_base + int64_t(2) * layer * a.slab_bytes) +
               (blk * a.page * a.hkv + h) * d;
  const int64_t row = int64_t(a.hkv) * d;
  float lo[IX_MAX_EPL], hi[IX_MAX_EPL];
#pragma unroll
  for (int i = 0; i < IX_MAX_EPL; ++i) {
    lo[i] = INFINITY;
    hi[i] = -INFINITY;
  }
#pragma unroll 4
  for (int r = 0; r < a.page; ++r) {
#pragma unroll
    for (int i = 0; i < IX_MAX_EPL; ++i) {
      const int e = lane + 32 * i;
      if (e < d) {
        const float x = to_f<T>(k[r * row + e]);
        lo[i] = fmin_nan(lo[i], x);
        hi[i] = fmax_nan(hi[i], x);
      }
    }
  }
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < IX_MAX_EPL; ++i)
    if (lane + 32 * i < d) top = fmax_nan(top, fmax_nan(fabsf(lo[i]), fabsf(hi[i])));
#pragma unroll
  for (int off = 16; off; off >>= 1) top = fmax_nan(top, __shfl_xor_sync(0xffffffffu, top, off));
  const float scale = __fmul_rn(top, 1.0f / 127.0f);
  const int64_t entry = (int64_t(layer) * a.num_blocks + blk) * a.hkv + h;
  int8_t* c = a.codes + entry * 2 * d;
#pragma unroll
  for (int i = 0; i < IX_MAX_EPL; ++i) {
    const int e = lane + 32 * i;
    if (e < d) {
      c[e] = code_of(lo[i], scale, false);
      c[d + e] = code_of(hi[i], scale, true);
    }
  }
  if (lane == 0) a.scales[entry] = scale;
}

// The same for heads of LPR 16-byte vectors (8, 16 or 32): LPR lanes on a key,
// 32 / LPR keys at a time, four loads in flight; a lane keeps VE dims.
template <typename T, int LPR>
__device__ __forceinline__ void index_entry_vec(const IndexArgs& a, int layer, int64_t blk, int h, int lane) {
  constexpr int VE = 16 / int(sizeof(T)), D = LPR * VE, RPI = 32 / LPR;
  const T* k = reinterpret_cast<const T*>(a.k_base + int64_t(2) * layer * a.slab_bytes) +
               (blk * a.page * a.hkv + h) * D + (lane % LPR) * VE;
  const int64_t row = int64_t(a.hkv) * D;
  // bounds as packed words: two 16-bit or one 32-bit value each
  uint4 mn{}, mx{};
  bool any = false;
  for (int r0 = lane / LPR; r0 < a.page; r0 += 4 * RPI) {
    uint4 x[4];
#pragma unroll
    for (int b = 0; b < 4; ++b)
      if (r0 + b * RPI < a.page) x[b] = *reinterpret_cast<const uint4*>(k + (r0 + b * RPI) * row);
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      if (r0 + b * RPI >= a.page) continue;
      mn = any ? min_words<T>(mn, x[b]) : x[b];
      mx = any ? max_words<T>(mx, x[b]) : x[b];
      any = true;
    }
  }
  // lanes without a key (fewer keys than lanes take) offer their neighbours nothing
#pragma unroll
  for (int off = LPR; off < 32; off <<= 1) {
    const uint4 on = shfl_xor4(mn, off), ox = shfl_xor4(mx, off);
    const bool there = __shfl_xor_sync(0xffffffffu, int(any), off) != 0;
    mn = !there ? mn : any ? min_words<T>(mn, on) : on;
    mx = !there ? mx : any ? max_words<T>(mx, ox) : ox;
    any |= there;
  }
  // every lane of a column holds its bounds now: the RPI lanes share the vector's words
  float top = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) top = fmax_nan(top, top_of_word<T>(word_of(mn, w), word_of(mx, w)));
#pragma unroll
  for (int off = 1; off < LPR; off <<= 1) top = fmax_nan(top, __shfl_xor_sync(0xffffffffu, top, off));
  const float scale = __fmul_rn(top, 1.0f / 127.0f);
  const int64_t entry = (int64_t(layer) * a.num_blocks + blk) * a.hkv + h;
  int8_t* out = a.codes + entry * 2 * D + (lane % LPR) * VE;
  constexpr int WPL = 4 / RPI;  // words a lane encodes
#pragma unroll
  for (int u = 0; u < WPL; ++u) {
    const int w = lane / LPR * WPL + u;
    store_codes<T>(out + w * (VE / 4), D, word_of(mn, w), word_of(mx, w), scale);
  }
  if (lane == 0) a.scales[entry] = scale;
}

// layer >= 0: one CTA per IX_TOKENS tokens; the pages whose last slot one of
// them fills are indexed, its warps taking the KV heads. layer < 0: one CTA per
// (block, layer). LPR 0: any head size.
constexpr int IX_TOKENS = 16;
template <typename T, int LPR>
__global__ void __launch_bounds__(256) page_index_kernel(const IndexArgs a) {
  auto index_one = [&](int layer, int64_t blk, int h, int ln) {
    if constexpr (LPR == 0) index_entry<T>(a, layer, blk, h, ln);
    else index_entry_vec<T, LPR>(a, layer, blk, h, ln);
  };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  pdl_trigger();
  pdl_wait();  // the keys were written by the append just before
  if (a.layer < 0) {
    const int64_t i = blockIdx.x / a.num_layers;
    const int layer = int(blockIdx.x % a.num_layers);
    const int64_t blk = a.ids[i];
    if (blk < 0 || blk >= a.num_blocks) {
      if (threadIdx.x == 0 && layer == 0) flag(a.st, PKV_DEV_SLOT_OOB);
      return;
    }
    for (int h = warp; h < a.hkv; h += nw) index_one(layer, blk, h, lane);
    return;
  }
  const int64_t t = int64_t(blockIdx.x) * IX_TOKENS + lane;
  const int64_t slot = lane < IX_TOKENS && t < a.n ? a.ids[t] : -1;
  // a slot outside the pool was flagged by the append
  const bool done = slot >= 0 && slot < a.num_blocks * a.page && slot % a.page == a.page - 1;
  uint32_t todo = __ballot_sync(0xffffffffu, done);
  while (todo) {
    const int l = __ffs(todo) - 1;
    todo &= todo - 1;
    const int64_t blk = __shfl_sync(0xffffffffu, slot, l) / a.page;
    for (int h = warp; h < a.hkv; h += nw) index_one(a.layer, blk, h, lane);
  }
}

template <typename T>
int launch_index(const IndexArgs& a, int64_t grid, cudaStream_t s) {
  // pool rows of whole 16-byte vectors (the base is 16-byte aligned): the vector forms
  const int lpr = (a.d * int(sizeof(T))) % 16 == 0 ? a.d * int(sizeof(T)) / 16 : 0;
  auto kern = lpr == 8 ? page_index_kernel<T, 8> : lpr == 16 ? page_index_kernel<T, 16>
              : lpr == 32 ? page_index_kernel<T, 32> : page_index_kernel<T, 0>;
  PKV_CUDA_RET(launch_kernel(kern, dim3(unsigned(grid)), dim3(unsigned(32 * std::min(a.hkv, 8))), 0, s, true, a));
  return PKV_OK;
}

int run_index(const pkv_pool& p, const pkv_page_index* ix, int layer, const int32_t* ids, int64_t n, int32_t* st,
              cudaStream_t s) {
  IndexArgs a;
  a.k_base = static_cast<const char*>(p.base);
  a.codes = ix->codes;
  a.scales = ix->scales;
  a.ids = ids;
  a.st = st;
  a.n = n;
  a.num_blocks = p.num_blocks;
  a.slab_bytes = slab_bytes(p);
  a.layer = layer;
  a.num_layers = p.num_layers;
  a.hkv = p.n_kv_heads;
  a.d = p.head_dim;
  a.page = p.block_size;
  const int64_t grid = layer >= 0 ? (n + IX_TOKENS - 1) / IX_TOKENS : n * p.num_layers;
  if (grid >= (int64_t(1) << 31)) return fail(PKV_ERR_ARG, "too many blocks for one call");
  switch (p.dtype) {
    case PKV_F16: return launch_index<__half>(a, grid, s);
    case PKV_BF16: return launch_index<__nv_bfloat16>(a, grid, s);
    default: return launch_index<float>(a, grid, s);
  }
}

template <typename T>
int launch_rope_append(const RopeAppendArgs& a, bool vec, bool inter, cudaStream_t s) {
  const int64_t warps = a.n_tokens * a.wpt;
  const int64_t grid = (warps * 32 + 255) / 256;
  if (grid >= (int64_t(1) << 31)) return fail(PKV_ERR_ARG, "too many tokens for one call");
  auto kern = vec ? (inter ? rope_append_kernel<T, true, true> : rope_append_kernel<T, true, false>)
                  : (inter ? rope_append_kernel<T, false, true> : rope_append_kernel<T, false, false>);
  PKV_CUDA_RET(launch_kernel(kern, dim3(unsigned(grid)), dim3(256), 0, s, true, a));
  return PKV_OK;
}

}  // namespace

int check_index(const pkv_pool& p, const pkv_page_index* ix) {
  if (!ix || !ix->codes || !ix->scales) return fail(PKV_ERR_ARG, "page index codes and scales must be non-NULL");
  if (reinterpret_cast<uintptr_t>(ix->codes) & 15) return fail(PKV_ERR_ARG, "page index codes must be 16-byte aligned");
  if (p.dtype != PKV_F16 && p.dtype != PKV_BF16 && p.dtype != PKV_F32)
    return fail(PKV_ERR_UNSUPPORTED, "the page index takes fp16, bf16 or fp32 pools");
  if (p.head_dim > 256) return fail(PKV_ERR_UNSUPPORTED, "the page index takes head_dim up to 256");
  return PKV_OK;
}

}  // namespace pkv

using namespace pkv;

extern "C" int pkv_page_index_update(const pkv_pool* pool, const pkv_page_index* index, int32_t layer,
                                     const int32_t* slot_mapping, int64_t n_tokens, int32_t* dev_status,
                                     void* stream) {
  if (int rc = check_pool(pool)) return rc;
  if (int rc = check_index(*pool, index)) return rc;
  if (layer < 0 || layer >= pool->num_layers)
    return fail(PKV_ERR_ARG, "layer_idx " + std::to_string(layer) + " out of range [0, " +
                                 std::to_string(pool->num_layers) + ")");
  if (n_tokens < 0) return fail(PKV_ERR_ARG, "n_tokens must be >= 0");
  if (n_tokens == 0) return PKV_OK;
  if (!slot_mapping) return fail(PKV_ERR_ARG, "slot_mapping must be non-NULL");
  return run_index(*pool, index, layer, slot_mapping, n_tokens, dev_status, static_cast<cudaStream_t>(stream));
}

extern "C" int pkv_page_index_rebuild(const pkv_pool* pool, const pkv_page_index* index, const int32_t* block_ids,
                                      int64_t nb, int32_t* dev_status, void* stream) {
  if (int rc = check_pool(pool)) return rc;
  if (int rc = check_index(*pool, index)) return rc;
  if (nb < 0) return fail(PKV_ERR_ARG, "nb must be >= 0");
  if (nb == 0) return PKV_OK;
  if (!block_ids) return fail(PKV_ERR_ARG, "block_ids must be non-NULL");
  return run_index(*pool, index, -1, block_ids, nb, dev_status, static_cast<cudaStream_t>(stream));
}

extern "C" int pkv_rope_append(const pkv_pool* pool, int32_t layer, const void* q, int64_t q_stride, void* q_out,
                               int32_t n_heads, const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                               const int32_t* slot_mapping, const int64_t* positions, int64_t n_tokens,
                               const float* rope_cos, const float* rope_sin, int64_t rope_max_pos,
                               int32_t rotary_dim, int32_t interleaved, const pkv_page_index* index,
                               int32_t* dev_status, void* stream) {
  if (int rc = check_pool(pool)) return rc;
  const pkv_pool& p = *pool;
  if (layer < 0 || layer >= p.num_layers)
    return fail(PKV_ERR_ARG, "layer_idx " + std::to_string(layer) + " out of range [0, " +
                                 std::to_string(p.num_layers) + ")");
  if (p.dtype != PKV_F16 && p.dtype != PKV_BF16 && p.dtype != PKV_F32)
    return fail(PKV_ERR_UNSUPPORTED, "pkv_rope_append takes fp16, bf16 or fp32 pools");
  if (index)
    if (int rc = check_index(p, index)) return rc;
  if (n_tokens < 0 || n_heads < 0) return fail(PKV_ERR_ARG, "n_tokens and n_heads must be >= 0");
  if (rotary_dim <= 0 || rotary_dim % 2 || rotary_dim > p.head_dim)
    return fail(PKV_ERR_ARG, "rotary_dim must be even and in [2, head_dim]");
  if (n_tokens == 0) return PKV_OK;
  if ((n_heads > 0 && (!q || !q_out)) || !k || !v || !slot_mapping || !positions || !rope_cos || !rope_sin)
    return fail(PKV_ERR_ARG, "q, q_out, k, v, slot_mapping, positions and the rope tables must be non-NULL");
  if (rope_max_pos <= 0) return fail(PKV_ERR_ARG, "rope_max_pos must be positive");
  const int es = elem_size(p.dtype);
  const int64_t qrow = int64_t(n_heads) * p.head_dim, krow = int64_t(p.n_kv_heads) * p.head_dim;
  if ((n_heads > 0 && q_stride < qrow) || k_stride < krow || v_stride < krow)
    return fail(PKV_ERR_ARG, "a token stride is smaller than the token's row");
  if (qrow + krow >= (int64_t(1) << 30)) return fail(PKV_ERR_ARG, "heads * head_dim too large");
  RopeAppendArgs a;
  a.q = static_cast<const char*>(q);
  a.k = static_cast<const char*>(k);
  a.v = static_cast<const char*>(v);
  a.q_out = static_cast<char*>(q_out);
  a.k_slab = static_cast<char*>(p.base) + int64_t(2) * layer * slab_bytes(p);
  a.v_slab = a.k_slab + slab_bytes(p);
  a.slots = slot_mapping;
  a.positions = positions;
  a.cs = rope_cos;
  a.sn = rope_sin;
  a.st = dev_status;
  a.q_stride = q_stride * es;
  a.k_stride = k_stride * es;
  a.v_stride = v_stride * es;
  a.qo_stride = qrow * es;
  a.n_tokens = n_tokens;
  a.n_slots = p.num_blocks * p.block_size;
  a.max_pos = rope_max_pos;
  a.hq = n_heads;
  a.hkv = p.n_kv_heads;
  a.d = p.head_dim;
  a.half = rotary_dim / 2;
  // 16-byte vectors where every row, head and column a unit touches is 16-byte aligned
  const int ve = 16 / es;
  uintptr_t al = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | uintptr_t(a.k_stride) |
                 uintptr_t(a.v_stride) | uintptr_t(int64_t(p.head_dim) * es) | reinterpret_cast<uintptr_t>(rope_cos) |
                 reinterpret_cast<uintptr_t>(rope_sin) | uintptr_t(slab_bytes(p));
  if (n_heads > 0)
    al |= reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out) | uintptr_t(a.q_stride);
  a.cols = 1;
  while (a.cols < a.half / ve) a.cols *= 2;
  const bool vec = (al & 15) == 0 && a.half % ve == 0 && a.cols <= 32;
  // one warp per token from eight tokens per SM on, else up to 8 (512 tokens of
  // 48 heads of 64: four warps 4.2 us, eight 6.5; 1700: one 8.4, four 10.3)
  const int64_t want = int64_t(num_sms()) * 8;
  a.wpt = n_tokens >= want ? 1 : (2 * n_tokens >= want ? 2 : (4 * n_tokens >= want ? 4 : 8));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool inter = interleaved != 0;
  int rc;
  switch (p.dtype) {
    case PKV_F16: rc = launch_rope_append<__half>(a, vec, inter, s); break;
    case PKV_BF16: rc = launch_rope_append<__nv_bfloat16>(a, vec, inter, s); break;
    default: rc = launch_rope_append<float>(a, vec, inter, s); break;
  }
  if (rc || !index) return rc;
  return run_index(p, index, layer, slot_mapping, n_tokens, dev_status, s);
}
