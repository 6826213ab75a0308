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
// One CTA per (query, KV head) does all of it: scores into shared memory, a
// radix selection over their order-preserving 32-bit keys, the listed pages
// ascending, then attention (S^T = K q^T and O^T += V^T P^T on 16-token tiles,
// fp32 online softmax) with the pages spread over its warps and merged at the
// end.
#include <algorithm>
#include <type_traits>

#include "pkv_common.cuh"

namespace pkv {
namespace {

struct SparseArgs {
  const void* q;
  void* out;
  int32_t* pages;        // [n_tokens][n_kv][budget], written by a selection, read otherwise
  const int8_t* codes;   // this layer's index entries [num_blocks][n_kv][2][d]
  const float* scales;   // [num_blocks][n_kv]
  const char* k_slab;
  const char* v_slab;
  const int32_t* cu_q;
  const int32_t* kv_lens;
  const int32_t* kv_indptr;
  const int32_t* kv_indices;
  const int32_t* last_page_len;
  const int32_t* batch_indices;
  int32_t* st;
  int64_t num_blocks, total_pages;
  int n_seqs, n_tokens, n_heads, n_kv, groups, d, page;
  int budget, sink, recent, max_pages;
  int mode;              // PKV_SPARSE_SELECT | PKV_SPARSE_ATTEND
  float scale_log2;
};

constexpr uint32_t KEY_FORCED = 0xffffffffu;  // first / last pages, always listed

// unsigned order = order of the scores; not a number above every number
__device__ __forceinline__ uint32_t score_key(float x) {
  if (x != x) return 0xfffffffeu;
  const uint32_t b = __float_as_uint(x + 0.f);  // -0 counts as 0
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// What a CTA works on: query t's sequence, its page list, its position.
struct Row {
  bool ok;
  int64_t pa;   // first entry of its page list
  int mine;     // page (of the list) that holds the query's own token
  int pos;      // the query's position
};
__device__ __forceinline__ Row find_row(const SparseArgs& a, int t) {
  Row r{false, 0, 0, 0};
  const int s = a.batch_indices[t];
  if (s < 0 || s >= a.n_seqs) return r;
  const int q0 = a.cu_q[s], q1 = a.cu_q[s + 1];
  const int64_t pa = a.kv_indptr[s], pb = a.kv_indptr[s + 1];
  const int lpl = a.last_page_len[s];
  const int64_t kv = (pb - pa - 1) * a.page + lpl;
  if (t < q0 || t >= q1 || pa < 0 || pb <= pa || pb > a.total_pages || lpl < 1 || lpl > a.page ||
      kv < q1 - q0 || kv >= 0x7fffffff || pb - pa > a.max_pages)
    return r;
  if (a.kv_lens && a.kv_lens[s] != kv) return r;
  r.ok = true;
  r.pa = pa;
  r.pos = int(kv) - (q1 - t);
  r.mine = r.pos / a.page;
  return r;
}

// q8 of the KV head's query heads into q8s [groups][2 d] (negative parts, then
// positive parts) and their scales into qs; one warp per head at a time.
template <typename T>
__device__ __forceinline__ void quantise_query(const SparseArgs& a, const T* q, int8_t* q8s, int stride, float* qs,
                                               int warp, int nw, int lane) {
  for (int g = warp; g < a.groups; g += nw) {
    const T* x = q + int64_t(g) * a.d;
    float top = 0.f;
    for (int e = lane; e < a.d; e += 32) top = fmaxf(top, fabsf(to_f<T>(x[e])));
#pragma unroll
    for (int off = 16; off; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    const float s = __fmul_rn(top, 1.0f / 127.0f);
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
  uint32_t hist[256];
  uint32_t wsum[2][32];
  uint32_t prefix, need, ties;
};

// The `budget` largest of keys[0..n) (n > budget), ties to the lowest index,
// into list[0..budget) ascending. Radix selection of the threshold, 8 bits a
// pass, ending as soon as a prefix holds exactly what is still needed, then one
// ordered compaction pass. All threads of the CTA call it.
__device__ __forceinline__ void select_top(const uint32_t* keys, int n, int budget, int* list, SelectSmem& sm) {
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5, nw = nt >> 5;
  uint32_t prefix = 0, mask = 0, need = budget;
  bool ties = true;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += nt) sm.hist[i] = 0;
    __syncthreads();
    for (int p = tid; p < n; p += nt) {
      const uint32_t k = keys[p];
      if ((k & mask) == prefix) atomicAdd(&sm.hist[(k >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (warp == 0) {  // lane l: bins 255 - 8 l .. 248 - 8 l
      uint32_t c[8], sum = 0;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        c[u] = sm.hist[255 - 8 * lane - u];
        sum += c[u];
      }
      uint32_t incl = sum;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += x;
      }
      const uint32_t before = incl - sum;
      if (before < need && incl >= need) {  // exactly one lane
        uint32_t above = before;
        int u = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (u == j && above + c[j] < need) {
            above += c[j];
            u = j + 1;
          }
        sm.prefix = prefix | (uint32_t(255 - 8 * lane - u) << shift);
        sm.need = need - above;
        sm.ties = (sm.hist[255 - 8 * lane - u] != need - above) ? 1u : 0u;
      }
    }
    __syncthreads();
    prefix = sm.prefix;
    need = sm.need;
    ties = sm.ties != 0;
    mask |= 0xffu << shift;
    if (!ties) break;
  }
  // listed: key above the threshold prefix, or (no excess ties) equal to it, or the first `need` equal ones
  uint32_t base_sel = 0, base_eq = 0;
  for (int p0 = 0; p0 < n; p0 += nt) {
    const int p = p0 + tid;
    const uint32_t k = p < n ? keys[p] & mask : 0u;
    const bool eq = p < n && k == prefix;
    bool sel = p < n && k > prefix;
    const uint32_t beq = __ballot_sync(0xffffffffu, eq);
    if (ties) {
      if (lane == 0) sm.wsum[0][warp] = __popc(beq);
      __syncthreads();
      uint32_t before = base_eq, all = 0;
      for (int w = 0; w < nw; ++w) {
        const uint32_t c = sm.wsum[0][w];
        if (w < warp) before += c;
        all += c;
      }
      base_eq += all;
      if (eq && before + __popc(beq & ((1u << lane) - 1u)) < need) sel = true;
    } else {
      sel = sel || eq;
    }
    const uint32_t b = __ballot_sync(0xffffffffu, sel);
    if (lane == 0) sm.wsum[1][warp] = __popc(b);
    __syncthreads();
    uint32_t before = base_sel, all = 0;
    for (int w = 0; w < nw; ++w) {
      const uint32_t c = sm.wsum[1][w];
      if (w < warp) before += c;
      all += c;
    }
    base_sel += all;
    if (sel) list[before + __popc(b & ((1u << lane) - 1u))] = p;
    __syncthreads();
  }
}

__device__ __forceinline__ bool forced_page(const SparseArgs& a, int p, int mine) {
  return p < a.sink || p > mine - a.recent;
}

// list[0..len): the query's pages, ascending (a given list: as given); writes
// the pages row of a selection. keys is scratch of n entries.
__device__ __forceinline__ int finish_list(const SparseArgs& a, uint32_t* keys, int n, int* list, int32_t* prow,
                                           SelectSmem& sm) {
  int len = n;
  if (n > a.budget) {
    select_top(keys, n, a.budget, list, sm);
    len = a.budget;
  } else {
    for (int p = threadIdx.x; p < n; p += blockDim.x) list[p] = p;
    __syncthreads();
  }
  for (int i = threadIdx.x; i < a.budget; i += blockDim.x) prow[i] = i < len ? list[i] : -1;
  return len;
}

__device__ __forceinline__ void imma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes global -> shared, or 16 zero bytes when !ok
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool ok) {
  const int n = ok ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// ---------------------------------------------------------------- 16-bit kernel
template <int D>
constexpr int sp_tps() { return D == 64 ? 2 : 1; }  // 16-token tiles per ring stage (8 KiB of K and V)
constexpr int SP_NST = 3;                            // ring stages per warp

template <int D, int NW>
constexpr size_t sp_ring_bytes() { return size_t(NW) * SP_NST * sp_tps<D>() * 2 * 16 * D * 2; }

template <typename T, int D, int NW>
__global__ void __launch_bounds__(NW * 32) sparse_kernel(const SparseArgs a) {
  constexpr int TPS = sp_tps<D>();
  constexpr int TILE = 16 * D * 2;       // bytes of one 16-token K or V tile
  constexpr int STAGE = TPS * 2 * TILE;
  constexpr int CH = D / 8;              // 16-byte chunks per row
  constexpr int KS = D / 16;             // 16-dim steps
  constexpr int Q8S = 2 * D + 16;
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char* ring = smem;                                      // aliases keys (scores end before the ring starts)
  uint32_t* keys = reinterpret_cast<uint32_t*>(smem);
  __shared__ int8_t q8s[8 * Q8S];
  __shared__ float qs[8];
  __shared__ SelectSmem sel;
  __shared__ float2 ml_all[NW][8];
  __shared__ int tile_valid[NW][SP_NST][TPS];  // visible tokens of each staged tile
  const size_t big = max(sp_ring_bytes<D, NW>(), (size_t(a.max_pages) * 4 + 15) & ~size_t(15));
  int* list = reinterpret_cast<int*>(smem + big);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c4 = lane & 3;
  const int t = int(blockIdx.x / unsigned(a.n_kv)), h = int(blockIdx.x % unsigned(a.n_kv));
  pdl_trigger();
  pdl_wait();  // q, the pool's new rows and the index may come from the kernels just before
  const Row row = find_row(a, t);
  const int G = a.groups;
  const int64_t q0 = (int64_t(t) * a.n_heads + int64_t(h) * G) * D;
  const T* q = static_cast<const T*>(a.q) + q0;
  T* out = static_cast<T*>(a.out) + q0;
  int32_t* prow = a.pages + (int64_t(t) * a.n_kv + h) * a.budget;
  if (!row.ok) {
    if (threadIdx.x == 0) flag(a.st, PKV_DEV_META_BAD);
    if (a.mode & PKV_SPARSE_SELECT)
      for (int i = threadIdx.x; i < a.budget; i += NW * 32) prow[i] = -1;
    if (a.mode & PKV_SPARSE_ATTEND)
      for (int i = threadIdx.x; i < G * D; i += NW * 32) out[i] = from_f<T>(0.f);
    return;
  }
  int len = a.budget;
  if (a.mode & PKV_SPARSE_SELECT) {
    const int n = row.mine + 1;
    if (n > a.budget) {
      for (int i = threadIdx.x; i < 8 * Q8S; i += NW * 32) q8s[i] = 0;
      if (threadIdx.x < 8) qs[threadIdx.x] = 0.f;
      __syncthreads();
      quantise_query<T>(a, q, q8s, Q8S, qs, warp, NW, lane);
      __syncthreads();
      // this lane's columns of B: head g, bytes 64 j + 16 c4 .. +15 of its 2 D
      constexpr int J = 2 * D / 64;
      uint4 b[J];
#pragma unroll
      for (int j = 0; j < J; ++j) b[j] = *reinterpret_cast<const uint4*>(q8s + g * Q8S + 64 * j + 16 * c4);
      const float s0 = qs[2 * c4], s1 = qs[2 * c4 + 1];
      const bool v0 = 2 * c4 < G, v1 = 2 * c4 + 1 < G;
      for (int p0 = warp * 32; p0 < n; p0 += NW * 32) {
        const int pl = p0 + lane;
        int id = pl < n ? a.kv_indices[row.pa + pl] : 0;
        const bool oob = id < 0 || id >= a.num_blocks;
        if (oob) {
          flag(a.st, PKV_DEV_SLOT_OOB);
          id = 0;
        }
        const float bs = a.scales[int64_t(id) * a.n_kv + h];
        // 4 rows of A per lane: pages g, g + 8, g + 16, g + 24 of the 32
        uint4 w[4][J];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int64_t idr = __shfl_sync(0xffffffffu, id, g + 8 * r);
          const uint4* src = reinterpret_cast<const uint4*>(a.codes + (idr * a.n_kv + h) * (2 * D)) + c4;
#pragma unroll
          for (int j = 0; j < J; ++j) w[r][j] = __ldg(src + 4 * j);
        }
        uint32_t mykey = 0;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          int acc[4] = {0, 0, 0, 0};
#pragma unroll
          for (int j = 0; j < J; ++j) {
            const uint4 &x = w[2 * half][j], &y = w[2 * half + 1][j];
            imma_s8(acc, x.x, y.x, x.y, y.y, b[j].x, b[j].y);
            imma_s8(acc, x.z, y.z, x.w, y.w, b[j].z, b[j].w);
          }
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float m = -INFINITY;
            if (v0) m = __fmul_rn(float(acc[2 * r]), s0);
            if (v1) m = fmaxf(m, __fmul_rn(float(acc[2 * r + 1]), s1));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
            // row g of (half, r) = page 16 half + 8 r + g: hand it to that lane
            const float mm = __shfl_sync(0xffffffffu, m, (lane & 7) * 4);
            if ((lane >> 3) == 2 * half + r) mykey = score_key(__fmul_rn(mm, bs));
          }
        }
        if (pl < n) keys[pl] = forced_page(a, pl, row.mine) ? KEY_FORCED : (oob ? 0u : mykey);
      }
      __syncthreads();
    }
    len = finish_list(a, keys, n, list, prow, sel);
  } else {
    for (int i = threadIdx.x; i < a.budget; i += NW * 32) list[i] = prow[i];
  }
  __syncthreads();
  if (!(a.mode & PKV_SPARSE_ATTEND)) return;

  // ---- attention over the listed pages, the tiles dealt to the warps in turn
  const int tpp = a.page / 16;
  const int n_tiles = len * tpp;
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
  const int n_stages = (n_tiles + TPS - 1) / TPS;
  const int mine_stages = n_stages > warp ? (n_stages - warp + NW - 1) / NW : 0;
  unsigned char* myring = ring + size_t(warp) * SP_NST * STAGE;
  const uint32_t ring0 = smem_u32(myring);
  const int64_t row_b = int64_t(a.n_kv) * D * 2;
  // valid tokens of tile i (0: not listed, past the query, outside the pool) and its block
  auto tile = [&](int i, int64_t& tok0) -> int {
    if (i >= n_tiles) return 0;
    const int p = list[i / tpp];
    if (p < 0 || p > row.mine) return 0;
    const int first = p * a.page + (i % tpp) * 16;
    if (first > row.pos) return 0;
    const int id = a.kv_indices[row.pa + p];
    if (id < 0 || id >= a.num_blocks) {
      flag(a.st, PKV_DEV_SLOT_OOB);
      return 0;
    }
    tok0 = int64_t(id) * a.page + (i % tpp) * 16;
    return min(16, row.pos - first + 1);
  };
  auto load = [&](int k) {  // this warp's k-th stage
    const uint32_t dst = ring0 + (k % SP_NST) * STAGE;
#pragma unroll
    for (int u = 0; u < TPS; ++u) {
      int64_t tok0 = 0;
      const int valid = tile((warp + k * NW) * TPS + u, tok0);
      if (lane == 0) tile_valid[warp][k % SP_NST][u] = valid;
#pragma unroll
      for (int c = 0; c < 16 * CH / 32; ++c) {
        const int idx = c * 32 + lane, r = idx / CH, ch = idx % CH;
        const int64_t off = (tok0 + r) * row_b + int64_t(h) * D * 2 + ch * 16;
        const bool ok = r < valid;  // rows past the query's position are never read: zeros
        const uint32_t sw = r * (D * 2) + ((ch ^ (r & 7)) << 4);
        cp_async16(dst + (2 * u) * TILE + sw, a.k_slab + (ok ? off : 0), ok);
        cp_async16(dst + (2 * u + 1) * TILE + sw, a.v_slab + (ok ? off : 0), ok);
      }
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
  for (int k = 0; k < SP_NST - 1; ++k) {
    if (k < mine_stages) load(k);
    cp_async_commit();
  }
  for (int k = 0; k < mine_stages; ++k) {
    if (k + SP_NST - 1 < mine_stages) load(k + SP_NST - 1);
    cp_async_commit();
    cp_async_wait<SP_NST - 1>();
    __syncwarp();
    const uint32_t src = ring0 + (k % SP_NST) * STAGE;
    float s[TPS][4];
    int valid[TPS];
#pragma unroll
    for (int u = 0; u < TPS; ++u) {
      valid[u] = tile_valid[warp][k % SP_NST][u];
#pragma unroll
      for (int e = 0; e < 4; ++e) s[u][e] = 0.f;
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int u = 0; u < TPS; ++u) {
        uint32_t af[4];
        const int chunk = 2 * ks + k_chk;
        ldsm_x4(af[0], af[1], af[2], af[3], src + (2 * u) * TILE + k_tok * (D * 2) + ((chunk ^ (k_tok & 7)) << 4));
        MmaOp<T>::run(s[u], af, qb[ks][0], qb[ks][1]);
      }
    float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
    for (int u = 0; u < TPS; ++u) {
      const bool a0 = g < valid[u], a1 = g + 8 < valid[u];
      s[u][0] = a0 ? s[u][0] * a.scale_log2 : -INFINITY;
      s[u][1] = a0 ? s[u][1] * a.scale_log2 : -INFINITY;
      s[u][2] = a1 ? s[u][2] * a.scale_log2 : -INFINITY;
      s[u][3] = a1 ? s[u][3] * a.scale_log2 : -INFINITY;
      x0 = fmaxf(x0, fmaxf(s[u][0], s[u][2]));
      x1 = fmaxf(x1, fmaxf(s[u][1], s[u][3]));
    }
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) {
      x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, off));
      x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, off));
    }
    const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
    const float al0 = ex2(m0 - n0), al1 = ex2(m1 - n1);
    m0 = n0;
    m1 = n1;
    float ls0 = 0.f, ls1 = 0.f;
    uint32_t pb[TPS][2];
#pragma unroll
    for (int u = 0; u < TPS; ++u) {
      const float p00 = ex2(s[u][0] - n0), p01 = ex2(s[u][1] - n1);
      const float p10 = ex2(s[u][2] - n0), p11 = ex2(s[u][3] - n1);
      ls0 += p00 + p10;
      ls1 += p01 + p11;
      pb[u][0] = movmatrix_t(MmaOp<T>::pack(p00, p01));
      pb[u][1] = movmatrix_t(MmaOp<T>::pack(p10, p11));
    }
    l0 = l0 * al0 + ls0;
    l1 = l1 * al1 + ls1;
#pragma unroll
    for (int mt = 0; mt < KS; ++mt) {
      o[mt][0] *= al0;
      o[mt][2] *= al0;
      o[mt][1] *= al1;
      o[mt][3] *= al1;
#pragma unroll
      for (int u = 0; u < TPS; ++u) {
        uint32_t af[4];
        const int chunk = 2 * mt + v_chk;
        ldsm_x4_t(af[0], af[1], af[2], af[3],
                  src + (2 * u + 1) * TILE + v_tok * (D * 2) + ((chunk ^ (v_tok & 7)) << 4));
        MmaOp<T>::run(o[mt], af, pb[u][0], pb[u][1]);
      }
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
  float* part = reinterpret_cast<float*>(ring);  // [NW][8][D + 4]
  constexpr int PS = D + 4;
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
    const float inv = L > 0.f ? 1.f / L : 0.f;  // nothing listed: zeros
    reinterpret_cast<uint32_t*>(out)[i] = L > 0.f || L != L ? MmaOp<T>::pack(y0 * inv, y1 * inv) : 0u;
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
  const Row row = find_row(a, t);
  const int64_t q0 = (int64_t(t) * a.n_heads + int64_t(h) * G) * D;
  const T* q = static_cast<const T*>(a.q) + q0;
  T* out = static_cast<T*>(a.out) + q0;
  int32_t* prow = a.pages + (int64_t(t) * a.n_kv + h) * a.budget;
  if (!row.ok) {
    if (threadIdx.x == 0) flag(a.st, PKV_DEV_META_BAD);
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
      quantise_query<T>(a, q, q8s, 2 * D, qs, warp, nw, lane);
      __syncthreads();
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
            best = fmaxf(best, __fmul_rn(float(dot), qs[g]));
          }
          key = score_key(__fmul_rn(best, a.scales[id * a.n_kv + h]));
        }
        if (lane == 0) keys[p] = forced_page(a, p, row.mine) ? KEY_FORCED : key;
      }
      __syncthreads();
    }
    len = finish_list(a, keys, n, list, prow, sel);
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

template <typename T, int D, int NW>
int launch_sparse_t(const SparseArgs& a, cudaStream_t s) {
  const size_t big = std::max(sp_ring_bytes<D, NW>(), (size_t(a.max_pages) * 4 + 15) & ~size_t(15));
  const size_t smem = big + size_t(a.budget) * 4;
  if (smem > SP_SMEM_MAX)
    return fail(PKV_ERR_UNSUPPORTED, "page lists of " + std::to_string(a.max_pages) + " pages with a budget of " +
                                         std::to_string(a.budget) + " do not fit in shared memory");
  auto kern = sparse_kernel<T, D, NW>;
  PKV_CUDA_RET(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(SP_SMEM_MAX)));
  PKV_CUDA_RET(launch_kernel(kern, dim3(unsigned(int64_t(a.n_tokens) * a.n_kv)), dim3(NW * 32), smem, s, true, a));
  return PKV_OK;
}

template <typename T>
int launch_sparse_generic(const SparseArgs& a, cudaStream_t s) {
  const size_t smem = size_t(a.max_pages) * 4 + size_t(a.budget) * 4 + size_t(a.groups) * (4 + 2 * a.d);
  if (smem > SP_SMEM_MAX)
    return fail(PKV_ERR_UNSUPPORTED, "page lists of " + std::to_string(a.max_pages) + " pages with a budget of " +
                                         std::to_string(a.budget) + " do not fit in shared memory");
  auto kern = sparse_generic_kernel<T>;
  PKV_CUDA_RET(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(SP_SMEM_MAX)));
  PKV_CUDA_RET(launch_kernel(kern, dim3(unsigned(int64_t(a.n_tokens) * a.n_kv)), dim3(256), smem, s, true, a));
  return PKV_OK;
}

template <typename T>
int launch_sparse(const SparseArgs& a, bool fast, cudaStream_t s) {
  if (!fast) return launch_sparse_generic<T>(a, s);
  return a.d == 64 ? launch_sparse_t<T, 64, 4>(a, s) : launch_sparse_t<T, 128, 4>(a, s);
}

}  // namespace



}  // namespace pkv

using namespace pkv;

extern "C" int pkv_attend_sparse(const pkv_pool* pool, const pkv_page_index* index, int32_t layer, int32_t n_heads,
                                 const void* q, void* out, int32_t* pages, float scale, int32_t budget, int32_t sink,
                                 int32_t recent, const pkv_batch* batch, const int32_t* batch_indices,
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
  if (!q || !pages || !batch_indices || ((mode & PKV_SPARSE_ATTEND) && !out))
    return fail(PKV_ERR_ARG, "q, out, pages and batch_indices must be non-NULL");
  if (!batch->cu_query_lens || !batch->kv_indptr || !batch->kv_last_page_len ||
      (batch->total_pages && !batch->kv_indices))
    return fail(PKV_ERR_ARG, "batch CSR pointers must be non-NULL");
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
  a.cu_q = batch->cu_query_lens;
  a.kv_lens = batch->kv_lens;
  a.kv_indptr = batch->kv_indptr;
  a.kv_indices = batch->kv_indices;
  a.last_page_len = batch->kv_last_page_len;
  a.batch_indices = batch_indices;
  a.st = batch->dev_status;
  a.num_blocks = p.num_blocks;
  a.total_pages = batch->total_pages;
  a.n_seqs = batch->n_seqs;
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
