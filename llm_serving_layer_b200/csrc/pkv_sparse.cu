// pkv_sparse.cu — page-sparse attention over the paged cache: each query scores
// the pages of its sequence with the page index, picks a budget of them per KV
// head and attends over their tokens only.
//
// Score of page p for one query and KV head with query heads g:
//   qs_g = max_d |q_gd| / 127,  q8_g = round(q_g / qs_g)          (int8)
//   I_g  = sum_d max(q8_gd lo8_pd, q8_gd hi8_pd)                  (whole number)
//   score = (max_g fl(I_g qs_g)) * bs_p
// lo8 / hi8 / bs: the page's index entry (pkv_append.cu). I_g is an upper bound
// of q8_g . k / bs for every key k of the page; being a sum of whole numbers it
// is the same in any order, and the two scalings are single rounded products,
// so the choice of pages is reproducible bit for bit. With q8 split into its
// negative and positive parts, I_g is one int8 dot product of 2 D entries,
// which the int8 tensor-core instruction takes 16 pages x 8 heads at a time.
//
// One row (query, KV head) is one CTA's, or a cluster's where rows are few:
// scores into shared memory, a selection over their order-preserving 32-bit keys,
// the listed pages ascending, then attention (S^T = K q^T and O^T += V^T P^T on
// 16-token tiles, fp32 online softmax) with the pages spread over its warps and
// merged at the end. One launch, nothing passes through global memory but the list.
//
// Bound by HBM once rows are many: 256 sequences of 1.4 to 4.1 k tokens, 64 pages
// each (2048 rows, fp16, 8 KV heads of 64): 537 MB of keys and values, 47 MB of
// index; the attention alone 92 us = 5.8 TB/s (0.90 of the copy rate), with the
// selection 108 us. Each row's chain (plan row, page ids, index entries,
// selection, page reads: about 11000 cycles before the first page is asked for)
// is hidden by the other CTAs of the SM there, and is the time itself where rows
// are few: 2048 pages of one sequence 12.8 us, of which the chain is two thirds.
#include <algorithm>
#include <mutex>
#include <string>
#include <type_traits>
#include <vector>

#include "pkv_common.cuh"

namespace pkv {
namespace {

struct Row;

struct SparseArgs {
  const void* q;
  void* out;
  int32_t* pages;        // [n_tokens][n_kv][budget], written by a selection, read otherwise
  const int8_t* codes;   // this layer's index entries [num_blocks][n_kv][2][d]
  const float* scales;   // [num_blocks][n_kv]
  const char* k_slab;
  const char* v_slab;
  const Row* rows;       // [n_tokens], the plan's
  const int32_t* kv_indices;
  int32_t* st;
  int64_t num_blocks;
  int n_tokens, n_heads, n_kv, groups, d, page;
  int budget, sink, recent, max_pages;
  int mode;              // PKV_SPARSE_SELECT | PKV_SPARSE_ATTEND
  float scale_log2;
};

// Scale of a query's codes from its largest magnitude: a query that is not finite
// has a NaN scale and codes 0, so that its scores are no numbers, all equal.
__device__ __forceinline__ float query_scale(float top) {
  return top < INFINITY ? __fmul_rn(top, 1.0f / 127.0f) : __int_as_float(0x7fffffff);
}

// unsigned order = order of the scores; not a number above every number
__device__ __forceinline__ uint32_t score_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.f);  // -0 counts as 0
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// What a CTA works on, one entry per query token, written by the plan: first
// entry of its sequence's page list, its position, and whether the step's tables
// are consistent for it (0: the row is zeros).
struct Row {
  int pa, pos, ok, unused;
};
static_assert(sizeof(Row) == sizeof(int4), "the plan's rows are int4");

struct RowArgs {
  const int32_t* cu_q;
  const int32_t* kv_lens;
  const int32_t* kv_indptr;
  const int32_t* last_page_len;
  const int32_t* batch_indices;
  int32_t* st;
  Row* rows;
  int64_t total_pages;
  int n_seqs, n_tokens, page, max_pages;
};
__global__ void __launch_bounds__(256) sparse_plan_kernel(const RowArgs a) {
  const int t = blockIdx.x * blockDim.x + threadIdx.x;
  if (t >= a.n_tokens) return;
  Row r{0, 0, 0, 0};
  const int s = a.batch_indices[t];
  if (s >= 0 && s < a.n_seqs) {
    const int q0 = a.cu_q[s], q1 = a.cu_q[s + 1];
    const int64_t pa = a.kv_indptr[s], pb = a.kv_indptr[s + 1];
    const int lpl = a.last_page_len[s];
    const int64_t kv = (pb - pa - 1) * a.page + lpl;
    if (t >= q0 && t < q1 && pa >= 0 && pb > pa && pb <= a.total_pages && lpl >= 1 && lpl <= a.page &&
        kv >= q1 - q0 && kv < 0x7fffffff && pb - pa <= a.max_pages && (!a.kv_lens || a.kv_lens[s] == kv)) {
      r.pa = int(pa);
      r.pos = int(kv) - (q1 - t);
      r.ok = 1;
    }
  }
  if (!r.ok) flag(a.st, PKV_DEV_META_BAD);
  a.rows[t] = r;
}

// q8 of the KV head's query heads into q8s [groups][2 d] (negative parts, then
// positive parts) and their scales into qs; one warp per head at a time.
template <typename T>
__device__ __forceinline__ void quantise_query(const SparseArgs& a, const T* q, int8_t* q8s, int stride, float* qs,
                                               int warp, int nw, int lane) {
  for (int g = warp; g < a.groups; g += nw) {
    const T* x = q + int64_t(g) * a.d;
    float top = 0.f;
    for (int e = lane; e < a.d; e += 32) top = fmax_nan(top, fabsf(to_f<T>(x[e])));
#pragma unroll
    for (int off = 16; off; off >>= 1) top = fmax_nan(top, __shfl_xor_sync(0xffffffffu, top, off));
    const float s = query_scale(top);
    for (int e = lane; e < a.d; e += 32) {
      float y = s > 0.f ? rintf(__fdiv_rn(to_f<T>(x[e]), s)) : 0.f;
      y = fminf(fmaxf(y, -127.f), 127.f);
      q8s[g * stride + e] = int8_t(fminf(y, 0.f));
      q8s[g * stride + a.d + e] = int8_t(fmaxf(y, 0.f));
    }
    if (lane == 0) qs[g] = s;
  }
}

struct SelectSmem {
  alignas(16) uint32_t hist[3][256];  // reversed bins: entry 255 - b counts bin b
  uint32_t cnt[2][32];                // per warp: keys above the threshold, keys equal to it
  uint32_t lo, hi;                    // range of the scored keys
};
static_assert(alignof(SelectSmem) >= alignof(uint4) && sizeof(SelectSmem::hist[0]) % sizeof(uint4) == 0,
              "select_top reads the bins four at a time");

// Before the scores: an empty range and histogram (a barrier follows).
__device__ __forceinline__ void select_init(SelectSmem& sm) {
  for (int i = threadIdx.x; i < 256; i += blockDim.x) sm.hist[0][i] = 0;
  if (threadIdx.x == 0) {
    sm.lo = 0xffffffffu;
    sm.hi = 0u;
  }
}
// Pages [f0, f1) of n are scored; the first and the last are listed anyway.
__device__ __forceinline__ int first_scored(const SparseArgs& a, int n) { return min(a.sink, n); }
__device__ __forceinline__ int end_scored(const SparseArgs& a, int n) { return max(min(a.sink, n), n - a.recent); }

// The query's `a.budget` pages out of n > budget: the unscored ones and the
// highest keys[p] of the others, ties to the lowest page; put(i, p) gets the
// i-th of them in ascending order. sm.lo / sm.hi hold the scored keys' range.
// Threshold search by 256-bin histograms over the keys' range (scores lie close
// together: equal-width bins over their range separate them in one or two
// passes, where fixed digits spend the first on common leading bits), until the
// threshold's bin is listed whole or holds one value: one barrier a pass, since
// every warp scans the bins itself. Then each warp counts and writes a
// contiguous share of the pages. All threads call it.
// KPT > 0: n <= 32 KPT keys per warp, which every lane reads once into registers.
template <int KPT, typename Put>
__device__ __forceinline__ void select_top(const SparseArgs& a, const uint32_t* keys, int n, SelectSmem& sm, Put put) {
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5, nw = nt >> 5;
  const int f0 = first_scored(a, n), f1 = end_scored(a, n);
  const int seg = (n + nw * 32 - 1) / (nw * 32) * 32;  // the warp's pages: [p0, p1)
  const int p0 = min(n, warp * seg), p1 = min(n, p0 + seg);
  uint32_t lo = sm.lo, hi = sm.hi;
  uint32_t need = uint32_t(a.budget - f0 - (n - f1));  // scored pages to list (fewer than there are)
  uint32_t held[KPT > 0 ? KPT : 1];
#pragma unroll
  for (int i = 0; i < KPT; ++i) {
    const int p = p0 + 32 * i + lane;
    held[i] = p < p1 ? keys[p] : 0u;
  }
  // f(page, key) over the lane's pages in order, 32 of the warp at a time (all lanes call it)
  auto each = [&](auto f) {
    if constexpr (KPT > 0) {
#pragma unroll
      for (int i = 0; i < KPT; ++i)
        if (p0 + 32 * i < p1) f(p0 + 32 * i + lane, held[i]);
    } else {
#pragma unroll 2
      for (int q = p0; q < p1; q += 32) f(q + lane, q + lane < p1 ? keys[q + lane] : 0u);
    }
  };
  int buf = 0;
  while (need > 0 && lo < hi) {
    const int shift = max(0, 24 - __clz(hi - lo));  // (hi - lo) >> shift < 256
    each([&](int p, uint32_t k) {
      if (p >= f0 && p < min(f1, p1) && k >= lo && k <= hi) atomicAdd(&sm.hist[buf][255 - ((k - lo) >> shift)], 1u);
    });
    // the next pass's bins, last read two passes ago: every warp has since met a barrier
    const int next = buf == 2 ? 0 : buf + 1;
    for (int i = tid; i < 256; i += nt) sm.hist[next][i] = 0;
    __syncthreads();
    // lane l: bins 255 - 8 l .. 248 - 8 l
    const uint4 x = reinterpret_cast<const uint4*>(sm.hist[buf])[2 * lane];
    const uint4 y = reinterpret_cast<const uint4*>(sm.hist[buf])[2 * lane + 1];
    const uint32_t c[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    const uint32_t sum = (x.x + x.y) + (x.z + x.w) + ((y.x + y.y) + (y.z + y.w));
    uint32_t incl = sum;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += v;
    }
    // the first lane whose bins reach `need`, then its first such bin
    const int src = __ffs(__ballot_sync(0xffffffffu, incl >= need)) - 1;
    uint32_t above = incl - sum, u = 0, cu = c[0];
#pragma unroll
    for (int v = 1; v < 8; ++v)
      if (u == uint32_t(v - 1) && above + cu < need) {
        above += cu;
        u = v;
        cu = c[v];
      }
    above = __shfl_sync(0xffffffffu, above, src);
    cu = __shfl_sync(0xffffffffu, cu, src);
    const uint32_t b = 255u - 8u * src - __shfl_sync(0xffffffffu, u, src);
    need -= above;
    const uint32_t top = lo + (((b + 1) << shift) - 1);  // wraps where the bin reaches past the last key
    const uint32_t bin_lo = lo + (b << shift);
    hi = min(hi, top < lo ? 0xffffffffu : top);
    lo = bin_lo;
    if (cu == need) break;  // every key of [lo, hi] is listed
    buf = next;
  }
  // listed: keys above hi, then `need` of those in [lo, hi] in page order (all of them, or they are equal)
  auto compare = [&](int p, uint32_t k, bool& gt, bool& eq) {
    gt = p < p1 && (p < f0 || p >= f1 || k > hi);
    eq = p < p1 && !gt && need > 0 && k >= lo;
  };
  uint32_t n_gt = 0, n_eq = 0;
  each([&](int p, uint32_t k) {
    bool gt, eq;
    compare(p, k, gt, eq);
    n_gt += __popc(__ballot_sync(0xffffffffu, gt));
    n_eq += __popc(__ballot_sync(0xffffffffu, eq));
  });
  if (lane == 0) {
    sm.cnt[0][warp] = n_gt;
    sm.cnt[1][warp] = n_eq;
  }
  __syncthreads();
  uint32_t eq_before = __reduce_add_sync(0xffffffffu, lane < warp ? sm.cnt[1][lane] : 0u);
  uint32_t at = __reduce_add_sync(0xffffffffu, lane < warp ? sm.cnt[0][lane] : 0u) + min(eq_before, need);
  each([&](int p, uint32_t k) {
    bool gt, eq;
    compare(p, k, gt, eq);
    const uint32_t beq = __ballot_sync(0xffffffffu, eq), below = (1u << lane) - 1u;
    const bool sel = gt || (eq && eq_before + __popc(beq & below) < need);
    const uint32_t b = __ballot_sync(0xffffffffu, sel);
    if (sel) put(int(at + __popc(b & below)), p);
    at += __popc(b);
    eq_before += __popc(beq);
  });
}

__device__ __forceinline__ void imma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// ---------------------------------------------------------------- 16-bit kernel
// Ring of one warp: NST stages of one 16-token K and V tile; reused for the
// warps' merge pieces.
template <int D, int NW, int NST>
constexpr size_t sp_ring_bytes() {
  constexpr size_t ring = size_t(NW) * NST * 2 * 16 * D * 2, merge = size_t(NW) * 8 * (D + 4) * 4;
  return ring > merge ? ring : merge;
}

// Thread-block clusters: a row's CTAs (1 when the launch has no cluster).
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
// address of this CTA's shared variable in the cluster's CTA `rank`
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void st_cluster(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void red_cluster_min(uint32_t addr, uint32_t v) {
  asm volatile("red.relaxed.cluster.shared::cluster.min.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void red_cluster_max(uint32_t addr, uint32_t v) {
  asm volatile("red.relaxed.cluster.shared::cluster.max.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t ld_cluster(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

// One row (query, KV head) per cluster of `cs` CTAs (1: no cluster): the CTAs
// share the row's scoring and its listed pages; rank 0 selects.
// SU: groups of 32 pages a warp scores at a time; MINB: CTAs per SM.
template <typename T, int D, int NW, int NST, int SU, int MINB>
__global__ void __launch_bounds__(NW * 32, MINB) sparse_kernel(const SparseArgs a, int cs) {
  constexpr int TILE = 16 * D * 2;       // bytes of one 16-token K or V tile
  constexpr int STAGE = 2 * TILE;
  constexpr int CH = D / 8;              // 16-byte chunks per row
  constexpr int KS = D / 16;             // 16-dim steps
  constexpr int Q8S = 2 * D + 16;
  constexpr int PS = D + 4;
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char* ring = smem;                          // aliases keys (scores end before the ring starts)
  uint32_t* keys = reinterpret_cast<uint32_t*>(smem);
  __shared__ __align__(16) int8_t q8s[8 * Q8S];
  __shared__ SelectSmem sel;
  __shared__ float2 ml_all[NW][8];
  __shared__ __align__(8) float2 ml_cta[8];
  __shared__ int tile_valid[NW][NST];               // visible tokens of each staged tile
  const size_t big = max(sp_ring_bytes<D, NW, NST>(), (size_t(a.max_pages) * 4 + 15) & ~size_t(15));
  int* list = reinterpret_cast<int*>(smem + big);      // pages within the sequence
  int* blks = list + a.budget;                         // their blocks (-1: outside the pool)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c4 = lane & 3;
  const uint32_t rank = cs > 1 ? cluster_rank() : 0u;
  const unsigned row_id = blockIdx.x / unsigned(cs);
  const int t = int(row_id / unsigned(a.n_kv)), h = int(row_id % unsigned(a.n_kv));
  pdl_trigger();
  pdl_wait();  // q, the pool's new rows and the index may come from the kernels just before
  const int4 row4 = __ldg(reinterpret_cast<const int4*>(a.rows + t));
  const int G = a.groups;
  const int64_t q0 = (int64_t(t) * a.n_heads + int64_t(h) * G) * D;
  const T* q = static_cast<const T*>(a.q) + q0;
  // this lane's part of the queries as the score products' B operand, loaded
  // while the row travels. Plain loads here and for the index: the kernel that writes
  // them may still run when this one starts, and the read-only path is for what
  // stays as it is from launch to end
  uint32_t qb[KS][2];
  if (g < G) {
    const T* qr = q + g * D + 2 * c4;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qb[ks][0] = *reinterpret_cast<const uint32_t*>(qr + ks * 16);
      qb[ks][1] = *reinterpret_cast<const uint32_t*>(qr + ks * 16 + 8);
    }
  } else {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qb[ks][0] = qb[ks][1] = 0u;
  }
  // (a plan made for longer lists than this call allows shared memory for is not followed)
  const struct { int64_t pa; int pos, mine; bool ok; } row{row4.x, row4.y, row4.y / a.page,
                                                           row4.z != 0 && row4.y / a.page < a.max_pages};
  T* out = static_cast<T*>(a.out) + q0;
  int32_t* prow = a.pages + (int64_t(t) * a.n_kv + h) * a.budget;
  if (!row.ok) {  // uniform over the cluster
    if (rank == 0) {
      if (a.mode & PKV_SPARSE_SELECT)
        for (int i = threadIdx.x; i < a.budget; i += NW * 32) prow[i] = -1;
      if (a.mode & PKV_SPARSE_ATTEND)
        for (int i = threadIdx.x; i < G * D; i += NW * 32) out[i] = from_f<T>(0.f);
    }
    return;
  }
  int len = a.budget;
  const int n = row.mine + 1;
  if ((a.mode & PKV_SPARSE_SELECT) && n > a.budget) {
    const int stride = cs * NW * 32 * SU;
    int p0 = (int(rank) * NW + warp) * 32 * SU, id[SU];
#pragma unroll
    for (int u = 0; u < SU; ++u) id[u] = p0 + 32 * u + lane < n ? a.kv_indices[row.pa + p0 + 32 * u + lane] : 0;
    // int8 query: the lanes (g, c4) hold head g's elements; the scale by a
    // maximum over the head's four lanes, the bytes through shared memory into
    // B's layout (head g, bytes 64 j + 16 c4 .. +15 of its 2 D)
    float top = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 x = unpack2<T>(qb[ks][e]);
        top = fmax_nan(top, fmax_nan(fabsf(x.x), fabsf(x.y)));
      }
    top = fmax_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmax_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const float q_scale = query_scale(top);
    select_init(sel);
    if (cs > 1) cluster_arrive();  // waited for before the first remote store
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if (ks % NW != warp) continue;  // the warps share the 16-dim steps
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 x = unpack2<T>(qb[ks][e]);
        int8_t* d8 = q8s + g * Q8S + ks * 16 + e * 8 + 2 * c4;
        float y0 = q_scale > 0.f ? rintf(__fdiv_rn(x.x, q_scale)) : 0.f;
        float y1 = q_scale > 0.f ? rintf(__fdiv_rn(x.y, q_scale)) : 0.f;
        y0 = fminf(fmaxf(y0, -127.f), 127.f);
        y1 = fminf(fmaxf(y1, -127.f), 127.f);
        *reinterpret_cast<char2*>(d8) = make_char2(int8_t(fminf(y0, 0.f)), int8_t(fminf(y1, 0.f)));
        *reinterpret_cast<char2*>(d8 + D) = make_char2(int8_t(fmaxf(y0, 0.f)), int8_t(fmaxf(y1, 0.f)));
      }
    }
    __syncthreads();
    constexpr int J = 2 * D / 64;
    uint4 b[J];
#pragma unroll
    for (int j = 0; j < J; ++j) b[j] = *reinterpret_cast<const uint4*>(q8s + g * Q8S + 64 * j + 16 * c4);
    // scales of this lane's columns, heads 2 c4 and 2 c4 + 1
    const float s0 = __shfl_sync(0xffffffffu, q_scale, 8 * c4), s1 = __shfl_sync(0xffffffffu, q_scale, 8 * c4 + 4);
    const bool v0 = 2 * c4 < G, v1 = 2 * c4 + 1 < G;
    const uint32_t keys0 = cs > 1 ? map_rank(smem_u32(keys), 0) : smem_u32(keys);
    if (cs > 1) cluster_wait();
    const int f0 = first_scored(a, n), f1 = end_scored(a, n);
    uint32_t lo = 0xffffffffu, hi = 0u;
    for (; p0 < n; p0 += stride) {
      // SU groups of 32 pages: all their index loads are in flight together
      uint4 w[SU][4][J];
      float bs[SU];
      bool oob[SU];
#pragma unroll
      for (int u = 0; u < SU; ++u) {
        oob[u] = id[u] < 0 || id[u] >= a.num_blocks;
        if (oob[u]) {
          flag(a.st, PKV_DEV_SLOT_OOB);
          id[u] = 0;
        }
        bs[u] = a.scales[int64_t(id[u]) * a.n_kv + h];
        // 4 rows of A per lane: pages g, g + 8, g + 16, g + 24 of the 32
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int64_t idr = __shfl_sync(0xffffffffu, id[u], g + 8 * r);
          const uint4* src = reinterpret_cast<const uint4*>(a.codes + (idr * a.n_kv + h) * (2 * D)) + c4;
#pragma unroll
          for (int j = 0; j < J; ++j) w[u][r][j] = src[4 * j];
        }
      }
#pragma unroll
      for (int u = 0; u < SU; ++u) {
        const int pn = p0 + stride + 32 * u + lane;
        id[u] = pn < n ? a.kv_indices[row.pa + pn] : 0;
      }
#pragma unroll
      for (int u = 0; u < SU; ++u) {
        const int pl = p0 + 32 * u + lane;
        uint32_t mykey = 0;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          int acc[4] = {0, 0, 0, 0};
#pragma unroll
          for (int j = 0; j < J; ++j) {
            const uint4 &x = w[u][2 * half][j], &y = w[u][2 * half + 1][j];
            imma_s8(acc, x.x, y.x, x.y, y.y, b[j].x, b[j].y);
            imma_s8(acc, x.z, y.z, x.w, y.w, b[j].z, b[j].w);
          }
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float m = -INFINITY;
            if (v0) m = __fmul_rn(float(acc[2 * r]), s0);
            if (v1) m = fmax_nan(m, __fmul_rn(float(acc[2 * r + 1]), s1));
            m = fmax_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = fmax_nan(m, __shfl_xor_sync(0xffffffffu, m, 2));
            // row g of (half, r) = page 16 half + 8 r + g: hand it to that lane
            const float mm = __shfl_sync(0xffffffffu, m, (lane & 7) * 4);
            if ((lane >> 3) == 2 * half + r) mykey = score_key(__fmul_rn(mm, bs[u]));
          }
        }
        if (oob[u]) mykey = 0u;
        if (pl >= f0 && pl < f1) {
          lo = min(lo, mykey);
          hi = max(hi, mykey);
        }
        if (pl < n) {
          if (cs > 1) st_cluster(keys0 + 4 * pl, mykey);
          else keys[pl] = mykey;
        }
      }
    }
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if (lane == 0 && lo <= hi) {  // this warp scored something: into rank 0's range
      if (cs > 1) {
        red_cluster_min(map_rank(smem_u32(&sel.lo), 0), lo);
        red_cluster_max(map_rank(smem_u32(&sel.hi), 0), hi);
      } else {
        atomicMin(&sel.lo, lo);
        atomicMax(&sel.hi, hi);
      }
    }
    if (cs > 1) {
      cluster_arrive();
      cluster_wait();
    } else {
      __syncthreads();
    }
  }
  // ---- the list: pages, their blocks (-1 for what is not attended)
  const bool attend = (a.mode & PKV_SPARSE_ATTEND) != 0;
  auto block_of = [&](int p) -> int {
    if (p < 0 || p > row.mine) return -1;
    const int id = a.kv_indices[row.pa + p];
    if (id >= 0 && id < a.num_blocks) return id;
    flag(a.st, PKV_DEV_SLOT_OOB);
    return -1;
  };
  if (a.mode & PKV_SPARSE_SELECT) {
    len = min(n, a.budget);
    if (n > a.budget) {
      if (rank == 0) {
        auto put = [&](int i, int p) {
          prow[i] = p;
          if (attend) list[i] = p;
        };
        if (n <= NW * 32 * 2) select_top<2>(a, keys, n, sel, put);
        else if (n <= NW * 32 * 8) select_top<8>(a, keys, n, sel, put);
        else select_top<0>(a, keys, n, sel, put);
      }
      if (cs > 1) {
        cluster_arrive();
        cluster_wait();  // rank 0's list is complete
        if (attend && rank > 0) {
          const uint32_t from = map_rank(smem_u32(list), 0);
          for (int i = threadIdx.x; i < len; i += NW * 32) list[i] = int(ld_cluster(from + 4 * i));
        }
      } else {
        __syncthreads();
      }
    } else {
      for (int i = threadIdx.x; i < a.budget; i += NW * 32) {
        if (rank == 0) prow[i] = i < n ? i : -1;
        if (i < n) list[i] = i;
      }
    }
  } else {
    for (int i = threadIdx.x; i < a.budget; i += NW * 32) list[i] = prow[i];
  }
  if (!attend) return;
  for (int i = threadIdx.x; i < len; i += NW * 32) blks[i] = block_of(list[i]);  // unselected lists: own entries
  __syncthreads();

  // ---- attention over the listed pages, the tiles dealt to the warps in turn
  const int tpp = a.page / 16;
  const int n_tiles = len * tpp;
  const int w0 = int(rank) * NW + warp, dw = cs * NW;  // this warp's tiles: w0, w0 + dw, ...
  const int my_tiles = n_tiles > w0 ? (n_tiles - w0 + dw - 1) / dw : 0;
  unsigned char* myring = ring + size_t(warp) * NST * STAGE;
  const uint32_t ring0 = smem_u32(myring);
  const int64_t row_b = int64_t(a.n_kv) * D * 2;
  const int r0 = lane / CH, ch = lane % CH;  // this lane's chunk of each row it copies
  const int64_t lane_off = int64_t(r0) * row_b + int64_t(h) * D * 2 + ch * 16;
  auto load = [&](int k) {  // this warp's k-th tile
    const uint32_t dst = ring0 + (k % NST) * STAGE;
    const int i = w0 + k * dw;
    const int e = tpp == 1 ? i : i / tpp, sub = tpp == 1 ? 0 : (i - e * tpp) * 16;
    const int blk = blks[e];
    const int valid = blk < 0 ? 0 : max(0, min(16, row.pos - (list[e] * a.page + sub) + 1));
    if (lane == 0) tile_valid[warp][k % NST] = valid;
    const int64_t off0 = (int64_t(blk) * a.page + sub) * row_b + lane_off;
#pragma unroll
    for (int c = 0; c < 16 * CH / 32; ++c) {
      const int r = c * (32 / CH) + r0;
      const bool ok = r < valid;  // rows past the query's position are never read: zeros
      const int64_t off = ok ? off0 + c * (32 / CH) * row_b : 0;
      const uint32_t sw = r * (D * 2) + ((ch ^ (r & 7)) << 4);
      cp_async16(dst + sw, a.k_slab + off, ok);
      cp_async16(dst + TILE + sw, a.v_slab + off, ok);
    }
  };
  float o[KS][4];
#pragma unroll
  for (int i = 0; i < KS; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
  float m0 = -1e30f, m1 = -1e30f, l0 = 0.f, l1 = 0.f;
  const int k_tok = lane & 15, k_chk = lane >> 4;
  const int v_tok = (lane & 7) + ((lane >> 4) << 3), v_chk = (lane >> 3) & 1;
#pragma unroll
  for (int k = 0; k < NST - 1; ++k) {
    if (k < my_tiles) load(k);
    cp_async_commit();
  }
  for (int k = 0; k < my_tiles; ++k) {
    if (k + NST - 1 < my_tiles) load(k + NST - 1);
    cp_async_commit();
    cp_async_wait<NST - 1>();
    __syncwarp();
    const uint32_t src = ring0 + (k % NST) * STAGE;
    const int valid = tile_valid[warp][k % NST];
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      uint32_t af[4];
      const int chunk = 2 * ks + k_chk;
      ldsm_x4(af[0], af[1], af[2], af[3], src + k_tok * (D * 2) + ((chunk ^ (k_tok & 7)) << 4));
      MmaOp<T>::run(s, af, qb[ks][0], qb[ks][1]);
    }
    const bool a0 = g < valid, a1 = g + 8 < valid;
    s[0] = a0 ? s[0] * a.scale_log2 : -INFINITY;
    s[1] = a0 ? s[1] * a.scale_log2 : -INFINITY;
    s[2] = a1 ? s[2] * a.scale_log2 : -INFINITY;
    s[3] = a1 ? s[3] * a.scale_log2 : -INFINITY;
    float x0 = fmaxf(s[0], s[2]), x1 = fmaxf(s[1], s[3]);
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) {
      x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, off));
      x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, off));
    }
    const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
    const float al0 = ex2(m0 - n0), al1 = ex2(m1 - n1);
    m0 = n0;
    m1 = n1;
    const float p00 = ex2(s[0] - n0), p01 = ex2(s[1] - n1);
    const float p10 = ex2(s[2] - n0), p11 = ex2(s[3] - n1);
    l0 = l0 * al0 + (p00 + p10);
    l1 = l1 * al1 + (p01 + p11);
    // P in the pool dtype, the product's operand type: relative 2^-11 (fp16) or 2^-8
    // (bf16) of weights that sum to 1 is that part of max |v| at most, as the
    // output's own rounding is; l sums them unrounded
    const uint32_t pb0 = movmatrix_t(MmaOp<T>::pack(p00, p01)), pb1 = movmatrix_t(MmaOp<T>::pack(p10, p11));
#pragma unroll
    for (int mt = 0; mt < KS; ++mt) {
      o[mt][0] *= al0;
      o[mt][2] *= al0;
      o[mt][1] *= al1;
      o[mt][3] *= al1;
      uint32_t af[4];
      const int chunk = 2 * mt + v_chk;
      ldsm_x4_t(af[0], af[1], af[2], af[3], src + TILE + v_tok * (D * 2) + ((chunk ^ (v_tok & 7)) << 4));
      MmaOp<T>::run(o[mt], af, pb0, pb1);
    }
    __syncwarp();  // every lane has read the stage before its slot is filled again
  }
  cp_async_wait<0>();
#pragma unroll
  for (int off = 4; off < 32; off <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, off);
    l1 += __shfl_xor_sync(0xffffffffu, l1, off);
  }
  // ---- merge of the warps' pieces (the ring is free once every warp is here)
  __syncthreads();
  float* part = reinterpret_cast<float*>(ring);  // [NW][8][PS]
  {
    float* mp = part + size_t(warp) * 8 * PS;
#pragma unroll
    for (int mt = 0; mt < KS; ++mt) {
      mp[(2 * c4) * PS + mt * 16 + g] = o[mt][0];
      mp[(2 * c4 + 1) * PS + mt * 16 + g] = o[mt][1];
      mp[(2 * c4) * PS + mt * 16 + g + 8] = o[mt][2];
      mp[(2 * c4 + 1) * PS + mt * 16 + g + 8] = o[mt][3];
    }
    if (g == 0) {
      ml_all[warp][2 * c4] = make_float2(m0, l0);
      ml_all[warp][2 * c4 + 1] = make_float2(m1, l1);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < G * D / 2; i += NW * 32) {
    const int hh = i / (D / 2), e = 2 * (i % (D / 2));
    float M = -1e30f;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, ml_all[w][hh].x);
    float L = 0.f, y0 = 0.f, y1 = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float c = ex2(ml_all[w][hh].x - M);
      const float2 v = *reinterpret_cast<const float2*>(part + (size_t(w) * 8 + hh) * PS + e);
      L += c * ml_all[w][hh].y;
      y0 += c * v.x;
      y1 += c * v.y;
    }
    if (cs == 1) {
      const float inv = L > 0.f ? 1.f / L : 0.f;  // nothing listed: zeros
      reinterpret_cast<uint32_t*>(out)[i] = L > 0.f || L != L ? MmaOp<T>::pack(y0 * inv, y1 * inv) : 0u;
    } else {  // this thread alone reads and writes these entries of warp 0's piece
      *reinterpret_cast<float2*>(part + size_t(hh) * PS + e) = make_float2(y0, y1);
      if (e == 0) ml_cta[hh] = make_float2(M, L);
    }
  }
  if (cs > 1) {
    // the CTAs' pieces, the output's elements shared among them
    cluster_arrive();
    cluster_wait();
    for (int i = int(rank) * NW * 32 + threadIdx.x; i < G * D / 2; i += cs * NW * 32) {
      const int hh = i / (D / 2), e = 2 * (i % (D / 2));
      const uint32_t ml = smem_u32(ml_cta + hh), pc = smem_u32(part + size_t(hh) * PS + e);
      float M = -1e30f;
      for (int r = 0; r < cs; ++r) M = fmaxf(M, ld_cluster2(map_rank(ml, r)).x);
      float L = 0.f, y0 = 0.f, y1 = 0.f;
      for (int r = 0; r < cs; ++r) {
        const float2 x = ld_cluster2(map_rank(ml, r)), v = ld_cluster2(map_rank(pc, r));
        const float c = ex2(x.x - M);
        L += c * x.y;
        y0 += c * v.x;
        y1 += c * v.y;
      }
      const float inv = L > 0.f ? 1.f / L : 0.f;
      reinterpret_cast<uint32_t*>(out)[i] = L > 0.f || L != L ? MmaOp<T>::pack(y0 * inv, y1 * inv) : 0u;
    }
    cluster_arrive();
    cluster_wait();  // no CTA leaves while another reads its pieces
  }
}

// ---------------------------------------------------------------- any geometry
// fp32 pools, other head sizes, page sizes or group sizes: the same steps on
// CUDA cores, one warp per page when scoring and per query head when attending.
constexpr int SG_MAX_DPL = 8;  // head_dim <= 256

template <typename T>
__global__ void __launch_bounds__(256) sparse_generic_kernel(const SparseArgs a) {
  extern __shared__ __align__(1024) unsigned char smem[];
  const int D = a.d, G = a.groups;
  uint32_t* keys = reinterpret_cast<uint32_t*>(smem);
  int* list = reinterpret_cast<int*>(keys + a.max_pages);
  float* qs = reinterpret_cast<float*>(list + a.budget);
  int8_t* q8s = reinterpret_cast<int8_t*>(qs + G);
  __shared__ SelectSmem sel;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  const int t = int(blockIdx.x / unsigned(a.n_kv)), h = int(blockIdx.x % unsigned(a.n_kv));
  pdl_trigger();
  pdl_wait();
  const int4 row4 = __ldg(reinterpret_cast<const int4*>(a.rows + t));
  // (a plan made for longer lists than this call allows shared memory for is not followed)
  const struct { int64_t pa; int pos, mine; bool ok; } row{row4.x, row4.y, row4.y / a.page,
                                                           row4.z != 0 && row4.y / a.page < a.max_pages};
  const int64_t q0 = (int64_t(t) * a.n_heads + int64_t(h) * G) * D;
  const T* q = static_cast<const T*>(a.q) + q0;
  T* out = static_cast<T*>(a.out) + q0;
  int32_t* prow = a.pages + (int64_t(t) * a.n_kv + h) * a.budget;
  if (!row.ok) {
    if (a.mode & PKV_SPARSE_SELECT)
      for (int i = threadIdx.x; i < a.budget; i += blockDim.x) prow[i] = -1;
    if (a.mode & PKV_SPARSE_ATTEND)
      for (int i = threadIdx.x; i < G * D; i += blockDim.x) out[i] = from_f<T>(0.f);
    return;
  }
  int len = a.budget;
  if (a.mode & PKV_SPARSE_SELECT) {
    const int n = row.mine + 1;
    if (n > a.budget) {
      select_init(sel);
      quantise_query<T>(a, q, q8s, 2 * D, qs, warp, nw, lane);
      __syncthreads();
      const int f0 = first_scored(a, n), f1 = end_scored(a, n);
      uint32_t lo = 0xffffffffu, hi = 0u;
      for (int p = warp; p < n; p += nw) {
        const int64_t id = a.kv_indices[row.pa + p];
        uint32_t key = 0u;
        if (id < 0 || id >= a.num_blocks) {
          if (lane == 0) flag(a.st, PKV_DEV_SLOT_OOB);
        } else {
          const int8_t* c = a.codes + (id * a.n_kv + h) * 2 * D;
          float best = -INFINITY;
          for (int g = 0; g < G; ++g) {
            int dot = 0;
            for (int e = lane; e < 2 * D; e += 32) dot += int(c[e]) * int(q8s[g * 2 * D + e]);
#pragma unroll
            for (int off = 16; off; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
            best = fmax_nan(best, __fmul_rn(float(dot), qs[g]));
          }
          key = score_key(__fmul_rn(best, a.scales[id * a.n_kv + h]));
        }
        if (lane == 0) keys[p] = key;
        if (p >= f0 && p < f1) {
          lo = min(lo, key);
          hi = max(hi, key);
        }
      }
      if (lane == 0 && lo <= hi) {
        atomicMin(&sel.lo, lo);
        atomicMax(&sel.hi, hi);
      }
      __syncthreads();
      select_top<0>(a, keys, n, sel, [&](int i, int p) { list[i] = p; });
    } else {
      for (int p = threadIdx.x; p < n; p += blockDim.x) list[p] = p;
    }
    len = min(n, a.budget);
    __syncthreads();
    for (int i = threadIdx.x; i < a.budget; i += blockDim.x) prow[i] = i < len ? list[i] : -1;
  } else {
    for (int i = threadIdx.x; i < a.budget; i += blockDim.x) list[i] = prow[i];
  }
  __syncthreads();
  if (!(a.mode & PKV_SPARSE_ATTEND)) return;

  const T* ks = reinterpret_cast<const T*>(a.k_slab);
  const T* vs = reinterpret_cast<const T*>(a.v_slab);
  const int64_t row_elems = int64_t(a.n_kv) * D;
  const int64_t keys_all = int64_t(len) * a.page;
  for (int g = warp; g < G; g += nw) {
    const T* qp = q + g * D;
    // row offset of key i of the listed pages, or -1
    auto key_row = [&](int64_t i) -> int64_t {
      const int p = list[i / a.page];
      if (p < 0 || p > row.mine || p * a.page + int(i % a.page) > row.pos) return -1;
      const int64_t id = a.kv_indices[row.pa + p];
      if (id < 0 || id >= a.num_blocks) {
        flag(a.st, PKV_DEV_SLOT_OOB);
        return -1;
      }
      return (id * a.page + i % a.page) * row_elems + int64_t(h) * D;
    };
    float m = -INFINITY, l = 0.f, acc[SG_MAX_DPL];
#pragma unroll
    for (int r = 0; r < SG_MAX_DPL; ++r) acc[r] = 0.f;
    for (int64_t i0 = 0; i0 < keys_all; i0 += 32) {
      const int64_t off = i0 + lane < keys_all ? key_row(i0 + lane) : -1;
      float sc = -INFINITY;
      if (off >= 0) {
        float dot = 0.f;
        for (int e = 0; e < D; ++e) dot += to_f<T>(qp[e]) * to_f<T>(ks[off + e]);
        sc = dot * a.scale_log2;
      }
      float cm = sc;
#pragma unroll
      for (int o = 16; o; o >>= 1) cm = fmaxf(cm, __shfl_xor_sync(0xffffffffu, cm, o));
      const float mn = fmaxf(m, cm);
      if (mn == -INFINITY) continue;  // nothing visible so far (uniform over the warp)
      const float al = exp2f(m - mn);
      const float p = exp2f(sc - mn);
      m = mn;
      float e = p;
#pragma unroll
      for (int o = 16; o; o >>= 1) e += __shfl_xor_sync(0xffffffffu, e, o);
      l = l * al + e;
#pragma unroll
      for (int r = 0; r < SG_MAX_DPL; ++r) acc[r] *= al;
      for (int kk = 0; kk < 32; ++kk) {
        const int64_t ro = __shfl_sync(0xffffffffu, off, kk);
        const float pk = __shfl_sync(0xffffffffu, p, kk);
        if (ro < 0) continue;
#pragma unroll
        for (int r = 0; r < SG_MAX_DPL; ++r) {
          const int d = lane + 32 * r;
          if (d < D) acc[r] += pk * to_f<T>(vs[ro + d]);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < SG_MAX_DPL; ++r) {
      const int d = lane + 32 * r;
      if (d < D) out[g * D + d] = from_f<T>(l == 0.f ? 0.f : acc[r] / l);
    }
  }
}

constexpr size_t SP_SMEM_MAX = 220 * 1024;  // dynamic part; the static part is below 7 KiB

// Raises a kernel's dynamic shared-memory limit once per device.
struct SmemReady {
  std::mutex mu;
  std::vector<char> done;
  int raise(const void* kern, int bytes) {
    int dev = 0;
    PKV_CUDA_RET(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lock(mu);
    if ((int)done.size() <= dev) done.resize(dev + 1, 0);
    if (!done[dev]) {
      PKV_CUDA_RET(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
      done[dev] = 1;
    }
    return PKV_OK;
  }
};

template <typename T, int D, int NW, int NST, int SU, int MINB>
int launch_sparse_t(const SparseArgs& a, int64_t rows, int cs, cudaStream_t s) {
  const size_t big = std::max(sp_ring_bytes<D, NW, NST>(), (size_t(a.max_pages) * 4 + 15) & ~size_t(15));
  const size_t smem = big + size_t(a.budget) * 8;
  if (smem > SP_SMEM_MAX)
    return fail(PKV_ERR_UNSUPPORTED, "page lists of " + std::to_string(a.max_pages) + " pages with a budget of " +
                                         std::to_string(a.budget) + " do not fit in shared memory");
  auto kern = sparse_kernel<T, D, NW, NST, SU, MINB>;
  static SmemReady ready;
  if (int rc = ready.raise(reinterpret_cast<const void*>(kern), int(SP_SMEM_MAX))) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(rows * cs));
  cfg.blockDim = dim3(NW * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cs > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim = {unsigned(cs), 1u, 1u};
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  PKV_CUDA_RET(cudaLaunchKernelEx(&cfg, kern, a, cs));
  return PKV_OK;
}

template <typename T>
int launch_sparse_generic(const SparseArgs& a, cudaStream_t s) {
  const size_t smem = size_t(a.max_pages) * 4 + size_t(a.budget) * 4 + size_t(a.groups) * (4 + 2 * a.d);
  if (smem > SP_SMEM_MAX)
    return fail(PKV_ERR_UNSUPPORTED, "page lists of " + std::to_string(a.max_pages) + " pages with a budget of " +
                                         std::to_string(a.budget) + " do not fit in shared memory");
  auto kern = sparse_generic_kernel<T>;
  static SmemReady ready;
  if (int rc = ready.raise(reinterpret_cast<const void*>(kern), int(SP_SMEM_MAX))) return rc;
  PKV_CUDA_RET(launch_kernel(kern, dim3(unsigned(int64_t(a.n_tokens) * a.n_kv)), dim3(256), smem, s, true, a));
  return PKV_OK;
}

template <typename T>
int launch_sparse(const SparseArgs& a, bool fast, cudaStream_t s) {
  if (!fast) return launch_sparse_generic<T>(a, s);
  // Rows are split over clusters of up to 8 CTAs while that leaves at most two CTAs
  // per SM: 8 rows of 2048 pages 34 us without, 13.4 with clusters of 8; 256 rows
  // of 350 pages 21 without, 27 in pairs.
  const int64_t rows = int64_t(a.n_tokens) * a.n_kv;
  const int sms = num_sms();
  int cs = 1;
  while (cs < 8 && rows * cs * 2 <= 2 * sms) cs *= 2;
  // head_dim 128: 8 KiB a tile and 152 registers leave two CTAs of 4 warps; 3 ring
  // stages 17.7 us on 140 rows of 250 pages, 2 stages 19.5, 4 stages 28.7
  if (a.d == 128) return launch_sparse_t<T, 128, 4, 3, 1, 2>(a, rows, cs, s);
  // Up to two CTAs per SM: 8 warps each (256 rows of 350 pages: 16.0 us, 4 warps
  // 20.5); more rows: 4 warps, five CTAs resident (2048 rows of 170 pages: 107 us,
  // four resident 116, 8 warps 127).
  if (rows * cs <= 2 * sms) return launch_sparse_t<T, 64, 8, 2, 1, 2>(a, rows, cs, s);
  return launch_sparse_t<T, 64, 4, 2, 1, 5>(a, rows, cs, s);
}

}  // namespace



}  // namespace pkv

using namespace pkv;

extern "C" int pkv_plan_sparse(const pkv_pool* pool, const pkv_batch* batch, const int32_t* batch_indices,
                               int32_t max_pages, void* rows, void* stream) {
  if (int rc = check_pool(pool)) return rc;
  if (!batch) return fail(PKV_ERR_ARG, "batch descriptor is NULL");
  if (batch->n_seqs <= 0) return fail(PKV_ERR_ARG, "batch has no sequences");
  if (batch->n_tokens < 0 || batch->total_pages < 0 || batch->total_pages >= (int64_t(1) << 31))
    return fail(PKV_ERR_ARG, "bad batch sizes");
  if (max_pages <= 0) return fail(PKV_ERR_ARG, "max_pages must be positive");
  if (batch->n_tokens == 0) return PKV_OK;
  if (!rows || !batch_indices || !batch->cu_query_lens || !batch->kv_indptr || !batch->kv_last_page_len)
    return fail(PKV_ERR_ARG, "rows, batch_indices and the batch CSR pointers must be non-NULL");
  if (reinterpret_cast<uintptr_t>(rows) & 15) return fail(PKV_ERR_ARG, "rows must be 16-byte aligned");
  RowArgs a;
  a.cu_q = batch->cu_query_lens;
  a.kv_lens = batch->kv_lens;
  a.kv_indptr = batch->kv_indptr;
  a.last_page_len = batch->kv_last_page_len;
  a.batch_indices = batch_indices;
  a.st = batch->dev_status;
  a.rows = static_cast<Row*>(rows);
  a.total_pages = batch->total_pages;
  a.n_seqs = batch->n_seqs;
  a.n_tokens = batch->n_tokens;
  a.page = pool->block_size;
  a.max_pages = max_pages;
  sparse_plan_kernel<<<unsigned((batch->n_tokens + 255) / 256), 256, 0, static_cast<cudaStream_t>(stream)>>>(a);
  PKV_CUDA_RET(cudaGetLastError());
  return PKV_OK;
}

extern "C" int pkv_attend_sparse(const pkv_pool* pool, const pkv_page_index* index, int32_t layer, int32_t n_heads,
                                 const void* q, void* out, int32_t* pages, float scale, int32_t budget, int32_t sink,
                                 int32_t recent, const pkv_batch* batch, const void* rows,
                                 int32_t max_pages, int32_t mode, void* stream) {
  if (int rc = check_pool(pool)) return rc;
  const pkv_pool& p = *pool;
  if (layer < 0 || layer >= p.num_layers)
    return fail(PKV_ERR_ARG, "layer_idx " + std::to_string(layer) + " out of range [0, " +
                                 std::to_string(p.num_layers) + ")");
  if (n_heads <= 0 || n_heads % p.n_kv_heads)
    return fail(PKV_ERR_ARG, "n_heads must be a positive multiple of n_kv_heads");
  if (mode <= 0 || (mode & ~(PKV_SPARSE_SELECT | PKV_SPARSE_ATTEND)))
    return fail(PKV_ERR_ARG, "mode must be PKV_SPARSE_SELECT, PKV_SPARSE_ATTEND or both");
  if (budget <= 0) return fail(PKV_ERR_ARG, "budget must be positive");
  if (mode & PKV_SPARSE_SELECT) {
    if (int rc = check_index(p, index)) return rc;
    if (sink < 0 || recent < 1 || int64_t(sink) + recent > budget)
      return fail(PKV_ERR_ARG, "sink >= 0, recent >= 1 and sink + recent <= budget are needed");
  }
  if (p.dtype != PKV_F16 && p.dtype != PKV_BF16 && p.dtype != PKV_F32)
    return fail(PKV_ERR_UNSUPPORTED, "page-sparse attention takes fp16, bf16 or fp32 pools");
  if (p.head_dim > 256) return fail(PKV_ERR_UNSUPPORTED, "page-sparse attention takes head_dim up to 256");
  if (!batch) return fail(PKV_ERR_ARG, "batch descriptor is NULL");
  if (batch->n_seqs <= 0) return fail(PKV_ERR_ARG, "batch has no sequences");
  if (batch->n_tokens < 0 || batch->total_pages < 0 || batch->total_pages >= (int64_t(1) << 31))
    return fail(PKV_ERR_ARG, "bad batch sizes");
  if (batch->n_tokens == 0) return PKV_OK;
  if (!q || !pages || !rows || !batch->kv_indices || ((mode & PKV_SPARSE_ATTEND) && !out))
    return fail(PKV_ERR_ARG, "q, out, pages, rows and kv_indices must be non-NULL");
  if (max_pages <= 0) return fail(PKV_ERR_ARG, "max_pages must be positive");
  if (int64_t(batch->n_tokens) * p.n_kv_heads >= (int64_t(1) << 31))
    return fail(PKV_ERR_ARG, "too many tokens for one call");
  SparseArgs a;
  a.q = q;
  a.out = out;
  a.pages = pages;
  a.codes = nullptr;
  a.scales = nullptr;
  if (mode & PKV_SPARSE_SELECT) {
    const int64_t entries = int64_t(layer) * p.num_blocks * p.n_kv_heads;
    a.codes = index->codes + entries * 2 * p.head_dim;
    a.scales = index->scales + entries;
  }
  a.k_slab = static_cast<const char*>(p.base) + int64_t(2) * layer * slab_bytes(p);
  a.v_slab = a.k_slab + slab_bytes(p);
  a.rows = static_cast<const Row*>(rows);
  a.kv_indices = batch->kv_indices;
  a.st = batch->dev_status;
  a.num_blocks = p.num_blocks;
  a.n_tokens = batch->n_tokens;
  a.n_heads = n_heads;
  a.n_kv = p.n_kv_heads;
  a.groups = n_heads / p.n_kv_heads;
  a.d = p.head_dim;
  a.page = p.block_size;
  a.budget = budget;
  a.sink = sink;
  a.recent = recent;
  a.max_pages = max_pages;
  a.mode = mode;
  a.scale_log2 = scale * 1.4426950408889634f;
  // the tensor-core kernel: 16-bit pools, head_dim 64 or 128, pages of whole
  // 16-token tiles, up to 8 query heads per KV head, 4-byte aligned q and out
  const bool fast = p.dtype != PKV_F32 && (p.head_dim == 64 || p.head_dim == 128) && p.block_size % 16 == 0 &&
                    a.groups <= 8 && ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 3) == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (p.dtype) {
    case PKV_F16: return launch_sparse<__half>(a, fast, s);
    case PKV_BF16: return launch_sparse<__nv_bfloat16>(a, fast, s);
    default: return launch_sparse_generic<float>(a, s);
  }
}
