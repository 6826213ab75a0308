// pkv_shared.cu — attention of a batch whose sequences share leading pages
// (families of the radix prefix cache: their block tables start with the same
// physical pages).
//
// The sequences of a batch come in groups; group g's sequences share their
// first n_g pages. For a row of group g with keys split into the shared prefix A
// and its own rest B,
//   out = (w_A O_A + w_B O_B) / (w_A + w_B),   w_X = l_X 2^(m_X - m),
// with O_X the normalised attention over X, m_X its score maximum (log2 units) and
// l_X its sum of 2^(s - m_X). All rows of a group see all of A, so A is one dense
// product of (rows of the group) x (keys of A) per KV head, read once:
//
//   shared_check_kernel  once per step: verifies that a group's page lists agree
//   shared_plan_kernel   once per step: the work items, the pieces each row
//                        merges, and the list of the one-token sequences' rest
//   shared_kernel        one persistent launch, three CTAs per SM, two roles:
//                        tiles  tcgen05 tiles of 128 rows (128 / G tokens of the
//                               group x the G query heads of a KV head) over a
//                               range of A's 64-key blocks, and the rest B of
//                               sequences with several new tokens (causal)
//                        stream one warp per KV head walks the pages of the rest
//                               B of sequences with one new token (mma.sync on
//                               16-key pages, as the decode kernel)
//                        each leaves pieces (O, m, l) in fp32
//   shared_merge_kernel  the pieces of a row -> out
//
// A's keys are read once per 128 rows instead of once per sequence: its
// 4 D flops per (row, key) are bound by the tensor cores and the exponentials,
// the rest by HBM. So the roles run side by side on every SM: some CTAs stream
// while the others compute, and the streaming CTAs take tiles when they are done.
// 256 sequences of up to 768 own tokens in 32 groups with prefixes of up to 512
// (fp16, 32 / 8 heads, 230 MB): 49 us = 4.6 TB/s; 256 of up to 512 on one prefix
// of 4096 (146 MB and 8.6 GFLOP in tiles): 44 us; 4 short ones on 1024: 11 us, two
// launches' latency.
#include <algorithm>
#include <mutex>
#include <string>
#include <type_traits>
#include <vector>

#include "pkv_tc.cuh"

namespace pkv {
namespace {

constexpr int SH_MINB = 3;          // CTAs per SM
// Slots of the K and of the V ring. A K slot is free when its S is computed, a
// period before the next S is; a V slot when its P V is, a period later: with
// three K slots and K loaded two blocks ahead of V both have two periods' time.
constexpr int SH_KST = 3, SH_VST = 2;
constexpr int SH_TMEM_COLS = 128;   // S in columns 0-63, O in 64-127
constexpr int SH_PIECES = 16384;    // tile piece rows the workspace holds at most (x n_heads x 264 bytes)
constexpr int SH_WARPS = TC_THREADS / 32;
constexpr int SH_SST = 3;                         // ring stages of a streaming warp
constexpr int SH_TILE = TC_P * TC_D * 2;          // one 16-token K or V tile of a head
constexpr int SH_STAGE = 2 * SH_TILE;
constexpr size_t SH_RING = size_t(SH_WARPS) * SH_SST * SH_STAGE;

// Rows (consecutive tokens) against a page range of one list.
struct ShEnt {
  int t0, nt;      // first token, tokens
  int pa;          // first entry of the page list
  int pg0, pg1;    // pages of the list
  int lim0;        // last key token t0 sees
  int causal;      // 1: token t0 + i sees i more keys
  int lpl;         // tokens in page pg1 - 1
  int base;        // first piece row (-1: the result goes straight to out)
  int splits;      // ranges the pages are cut into
  int tiles;
  int item0;       // first item
};

// A work item of the tile role, without its KV head.
struct ShItem {
  int t0, nt;        // first token, tokens of the tile
  int pg_at, n_pg;   // first entry in kv_indices, pages of the range
  int nblk;          // 64-key blocks
  int lim0, causal;  // last key (counted from the range's first) the first token sees; 1: token i sees i more
  int tail_pg, lpl;  // page of the range with only lpl written tokens (-1: none)
  int piece;         // piece row of the first token (-1: straight to out)
  int h, zero;       // (published) KV head; a page id outside the pool: the item's rows are zeros
};
static_assert(sizeof(ShItem) == 3 * sizeof(int4), "items are read as three int4");

struct ShCtl {
  int n_items;
  int claim[2];    // items claimed, CTAs finished
  int n_stream;    // CTAs that stream first
  int n_ranges;    // ranges the listed pages are cut into (one warp per range and KV head)
  int listed;      // pages listed
};

struct ShLayout {
  size_t ctl, rows, list, seq_np, group_bad, ents, items, desc, fold, rest, part_o, part_ml, total;
  int64_t pieces, items_cap, slots;
};

inline size_t al256(size_t x) { return (x + 255) & ~size_t(255); }

int split_cap(int n_tokens) { return std::max(1, std::min(64, 4096 / std::max(n_tokens, 1))); }

// Ranges of the listed pages there can be: every warp of the launch streaming.
int max_ranges(int n_kv) { return SH_MINB * num_sms() * SH_WARPS / n_kv; }

ShLayout sh_layout(int n_heads, int n_kv, int n_seqs, int n_tokens, int64_t total_pages) {
  ShLayout w;
  size_t off = 0;
  const int cap = split_cap(n_tokens);
  const int tpt = TC_ROWS / std::max(1, std::min(8, n_heads / n_kv));
  w.pieces = std::min<int64_t>(int64_t(2) * n_tokens * cap, SH_PIECES);
  // every entity's last tile may be partial; an entity is a group or a sequence
  w.items_cap = (int64_t(2) * ((n_tokens + tpt - 1) / tpt) + 2 * int64_t(n_seqs)) * cap;
  // piece rows: the tiles', then one per (range, sequence) a streaming warp meets
  w.slots = w.pieces + n_seqs + max_ranges(n_kv);
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off = al256(off + bytes);
    return at;
  };
  w.ctl = take(sizeof(ShCtl));
  w.rows = take(sizeof(int32_t) * n_seqs);
  w.list = take(sizeof(int2) * n_seqs);
  w.seq_np = take(sizeof(int32_t) * n_seqs);
  w.group_bad = take(sizeof(int32_t) * n_seqs);
  w.ents = take(sizeof(ShEnt) * 2 * n_seqs);
  w.items = take(sizeof(ShItem) * w.items_cap);
  w.desc = take(sizeof(int2) * size_t(std::max<int64_t>(total_pages, 1)));
  w.fold = take(sizeof(int4) * std::max(n_tokens, 1));
  w.rest = take(sizeof(int4) * std::max(n_tokens, 1));
  w.part_o = take(sizeof(float) * size_t(w.slots) * n_heads * TC_D);
  w.part_ml = take(sizeof(float2) * size_t(w.slots) * n_heads);
  w.total = off;
  return w;
}

// ---------------------------------------------------------------- plan
struct PlanArgs {
  const int32_t* cu_q;
  const int32_t* kv_lens;
  const int32_t* kv_indptr;
  const int32_t* kv_indices;
  const int32_t* last_page_len;
  const int32_t* group_indptr;  // [n_groups + 1] over the sequences
  const int32_t* prefix_pages;  // [n_groups]
  int32_t* st;
  int64_t num_blocks, total_pages;
  int n_seqs, n_tokens, n_groups, page, n_kv, tpt, sms, splits_cap, grid;  // page: TC_P but for the check alone
  int64_t pieces_cap, items_cap;
  ShCtl* ctl;
  int32_t* rows;   // row of each listed one-token sequence
  int2* list;      // its first page in the list, its pages
  int32_t* seq_np; // shared pages of each sequence
  int32_t* group_bad;
  ShEnt* ents;
  ShItem* items;
  int2* desc;      // listed page {block, index of its sequence in the list << 7 | first << 6 | last << 5 | tokens}
  int4* fold;      // a row's pieces over the shared keys {first piece row, pieces, stride}
  int4* rest;      // ... over its own; {0, 0, 0, 1}: the tiles write the row; {0, 0, 0, 0}: nobody does
};

struct SeqInfo {
  bool ok;
  int q0, ql, pa, pages, lpl;
  int64_t kv;
};
__device__ __forceinline__ SeqInfo seq_info(const PlanArgs& a, int s) {
  SeqInfo r;
  r.q0 = a.cu_q[s];
  r.ql = a.cu_q[s + 1] - r.q0;
  const int64_t pa = a.kv_indptr[s], pb = a.kv_indptr[s + 1];
  r.lpl = a.last_page_len[s];
  r.pa = int(pa);
  r.pages = int(pb - pa);
  r.kv = (pb - pa - 1) * a.page + r.lpl;
  r.ok = r.q0 >= 0 && r.ql >= 1 && int64_t(r.q0) + r.ql <= a.n_tokens && pa >= 0 && pb > pa && pb <= a.total_pages &&
         r.lpl >= 1 && r.lpl <= a.page && r.kv >= r.ql && r.kv < 0x7fffffff && (!a.kv_lens || a.kv_lens[s] == r.kv);
  return r;
}
// group of sequence s: the last g with group_indptr[g] <= s
__device__ __forceinline__ int group_of(const PlanArgs& a, int s) {
  int lo = 0, hi = a.n_groups - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.group_indptr[mid] <= s) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// CTAs that stream first at the least, from the streaming's and the tiles' time on
// the whole GPU (a page of one KV head is 4 KiB at the copy rate; a block of a
// tile keeps its SM for 860 cycles): 7/4 an SM from four times the tiles' time on,
// below that the streaming's share, one an SM at most (256 sequences of 2 tokens
// on an 8192-token prefix: 7 CTAs, 46 us; one an SM 54).
__device__ __forceinline__ int stream_least(const PlanArgs& a, int listed, float blocks) {
  const float t_stream = float(listed) * a.n_kv * 4096.f / 6.4e6f, t_tiles = blocks * a.n_kv / a.sms * 0.45f;  // us
  if (t_stream >= 4.f * t_tiles) return a.sms * 7 / 4;
  return min(a.sms, int(a.grid * t_stream / (t_stream + t_tiles)) + 1);
}

// One CTA per sequence: do its leading pages agree with its group's first
// sequence's, and do its new tokens lie after them? If not the group is marked
// (where there are marks) and flagged, and computed without sharing.
__global__ void __launch_bounds__(128) shared_check_kernel(const PlanArgs a) {
  const int s = blockIdx.x;
  const int g = group_of(a, s);
  const int f = a.group_indptr[g], e = a.group_indptr[g + 1];
  const int np = a.prefix_pages[g];
  bool bad = f < 0 || s < f || s >= e || e > a.n_seqs || np < 0;
  if (!bad && np > 0) {
    const SeqInfo x = seq_info(a, s), y = seq_info(a, f);
    bad = !x.ok || !y.ok || int64_t(np) * a.page > x.kv - x.ql || np > y.pages;
    if (!bad)
      for (int i = threadIdx.x; i < np; i += blockDim.x) {
        const int id = a.kv_indices[x.pa + i];
        bad |= id != a.kv_indices[y.pa + i] || id < 0 || id >= a.num_blocks;
      }
  }
  if (bad) {
    flag(a.st, PKV_DEV_META_BAD);
    if (a.group_bad && g >= 0 && g < a.n_groups) a.group_bad[g] = 1;
  }
}

__global__ void __launch_bounds__(1024) shared_plan_kernel(const PlanArgs a) {
  __shared__ int warp_sum[32];
  __shared__ int s_bad, s_maxblk, s_tot, s_listed;
  __shared__ unsigned long long s_best;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    s_bad = (a.cu_q[0] != 0 || a.cu_q[a.n_seqs] != a.n_tokens || a.group_indptr[0] != 0 ||
             a.group_indptr[a.n_groups] != a.n_seqs) ? 1 : 0;
    *a.ctl = ShCtl{};
  }
  for (int t = tid; t < a.n_tokens; t += blockDim.x) a.fold[t] = a.rest[t] = make_int4(0, 0, 0, 0);
  __syncthreads();
  if (s_bad) {
    if (tid == 0) flag(a.st, PKV_DEV_META_BAD);
    __threadfence();
    return;
  }
  // share = 1: as the groups say. Should even one piece per row and range not
  // fit the workspace, a second round (share = 0) computes every sequence by itself.
  int n_ents = 0, chunk = 1, n_lo = 0;
  for (int share = 1; share >= 0; --share) {
    if (tid == 0) {
      s_maxblk = 1;
      s_listed = 0;
    }
    __syncthreads();
    for (int s = tid; s < a.n_seqs; s += blockDim.x) {
      const int g = group_of(a, s);
      const int f = a.group_indptr[g], e = a.group_indptr[g + 1];
      // a group of one sequence shares nothing
      const int np = share && e - f >= 2 && !a.group_bad[g] ? a.prefix_pages[g] : 0;
      a.seq_np[s] = np;
      if (a.cu_q[s + 1] - a.cu_q[s] == 1) atomicAdd(&s_listed, max(0, a.kv_indptr[s + 1] - a.kv_indptr[s] - np));
    }
    __syncthreads();
    // ---- entities: the shared groups, then the several-token sequences
    n_ents = 0;
    for (int c0 = 0; c0 < a.n_groups; c0 += blockDim.x) {
      const int g = c0 + tid;
      ShEnt x{};
      int is = 0;
      if (g < a.n_groups) {
        const int f = a.group_indptr[g], e = a.group_indptr[g + 1];
        const int np = f < e && f >= 0 && e <= a.n_seqs ? a.seq_np[f] : 0;
        if (np > 0) {
          is = 1;
          x.t0 = a.cu_q[f];
          x.nt = a.cu_q[e] - x.t0;
          x.pa = a.kv_indptr[f];
          x.pg0 = 0;
          x.pg1 = np;
          x.lim0 = np * TC_P - 1;
          x.lpl = TC_P;
          x.tiles = (x.nt + a.tpt - 1) / a.tpt;
          atomicMax(&s_maxblk, (np + TC_PPB - 1) / TC_PPB);
        }
      }
      int tot;
      const int i = n_ents + block_excl_scan(is, warp_sum, &tot);
      if (is) a.ents[i] = x;
      n_ents += tot;
    }
    for (int c0 = 0; c0 < a.n_seqs; c0 += blockDim.x) {
      const int s = c0 + tid;
      ShEnt x{};
      int is = 0;
      if (s < a.n_seqs) {
        const SeqInfo q = seq_info(a, s);
        if (!q.ok) {
          flag(a.st, PKV_DEV_META_BAD);
        } else if (q.ql > 1) {
          is = 1;
          x.t0 = q.q0;
          x.nt = q.ql;
          x.pa = q.pa;
          x.pg0 = a.seq_np[s];
          x.pg1 = q.pages;
          x.lim0 = int(q.kv) - q.ql;
          x.causal = 1;
          x.lpl = q.lpl;
          x.tiles = (x.nt + a.tpt - 1) / a.tpt;
          x.base = x.pg0 > 0 ? 0 : -1;
          if (x.pg0 > 0) atomicMax(&s_maxblk, (x.pg1 - x.pg0 + TC_PPB - 1) / TC_PPB);
        }
      }
      int tot;
      const int i = n_ents + block_excl_scan(is, warp_sum, &tot);
      if (is) a.ents[i] = x;
      n_ents += tot;
    }
    __threadfence_block();
    __syncthreads();
    // ---- blocks per range: each thread weighs one length. The CTAs that start
    // with tiles take an item after the other: rounds of a range's blocks and an
    // item's set-up and epilogue (four blocks' time); then the pieces, whose writing
    // and reading is three blocks' work for a full tile, and the merge's rounds of
    // eight. (256 sequences on a 4096-token prefix, 512-token rest: ranges of 16
    // blocks, 256 items, 44 us; 22 blocks 49, 32 blocks 57. 24 groups of 2 on
    // prefixes of up to 4000 tokens: 39 us, with a set-up of two blocks 53.)
    const int maxblk = s_maxblk;
    const int step = (maxblk + int(blockDim.x) - 1) / int(blockDim.x);
    const int cand = min(maxblk, (tid + 1) * step);
    float n_it = 0.f, rows = 0.f, n_blk = 0.f;
    int most = 1;
    int64_t pieces = 0;
    bool fits = true;
    for (int i = 0; i < n_ents; ++i) {
      const ShEnt x = a.ents[i];
      const int nb = (x.pg1 - x.pg0 + TC_PPB - 1) / TC_PPB;
      const int sp = x.base < 0 ? 1 : (nb + cand - 1) / cand;
      fits &= sp <= a.splits_cap;
      n_it += float(x.tiles) * sp;
      n_blk += float(x.tiles) * nb;
      if (x.base >= 0) {
        pieces += int64_t(x.nt) * sp;
        rows += float(x.nt) * sp;
        most = max(most, sp);
      }
    }
    fits &= pieces <= a.pieces_cap;
    n_lo = stream_least(a, s_listed, n_blk);
    const float slots = float(a.grid - n_lo), items = n_it * a.n_kv;
    const float est = ceilf(items / slots) * (cand + 4.f) + rows / a.tpt * a.n_kv * 3.f / a.sms + 1.5f * ((most + 7) / 8);
    if (tid == 0) s_best = ~0ull;
    __syncthreads();
    if (fits && (tid == 0 || (tid + 1) * step < maxblk + step))
      atomicMin(&s_best, (static_cast<unsigned long long>(__float_as_uint(est)) << 32) | unsigned(cand));
    __syncthreads();
    const unsigned long long best = s_best;
    __syncthreads();
    chunk = int(best & 0xffffffffu);
    if (best != ~0ull) break;  // always in the second round: nothing is shared, no pieces
  }
  // ---- piece rows and items of each entity
  int base0 = 0, item0 = 0;
  for (int c0 = 0; c0 < n_ents; c0 += blockDim.x) {
    const int i = c0 + tid;
    ShEnt x{};
    int np = 0, ni = 0;
    if (i < n_ents) {
      x = a.ents[i];
      const int nb = (x.pg1 - x.pg0 + TC_PPB - 1) / TC_PPB;
      x.splits = x.base < 0 ? 1 : (nb + chunk - 1) / chunk;
      np = x.base < 0 ? 0 : x.nt * x.splits;
      ni = x.tiles * x.splits;
    }
    int tp, ti;
    const int b = base0 + block_excl_scan(np, warp_sum, &tp);
    const int it = item0 + block_excl_scan(ni, warp_sum, &ti);
    if (i < n_ents) {
      if (x.base >= 0) x.base = b;
      x.item0 = it;
      a.ents[i] = x;
    }
    base0 += tp;
    item0 += ti;
  }
  __threadfence_block();
  __syncthreads();
  if (tid == 0) s_tot = item0 <= a.items_cap ? 1 : 0;
  __syncthreads();
  const bool room = s_tot != 0;  // the capacity covers every case: kept as a check
  for (int i = warp; room && i < n_ents; i += 32) {
    const ShEnt x = a.ents[i];
    for (int k = lane; k < x.tiles * x.splits; k += 32) {
      const int i0 = k / x.splits * a.tpt, sp = k % x.splits;
      ShItem I{};
      I.t0 = x.t0 + i0;
      I.nt = min(a.tpt, x.nt - i0);
      const int first = x.pg0 + (x.base < 0 ? 0 : sp * chunk * TC_PPB);
      const int last = x.base < 0 ? x.pg1 : min(x.pg1, first + chunk * TC_PPB);
      I.pg_at = x.pa + first;
      I.lim0 = x.lim0 + x.causal * i0 - first * TC_P;
      I.causal = x.causal;
      const int seen = I.lim0 + x.causal * (I.nt - 1);  // last key any of its rows sees
      I.n_pg = seen < 0 ? 0 : min(last - first, seen / TC_P + 1);
      I.nblk = max(1, (I.n_pg + TC_PPB - 1) / TC_PPB);  // a range no row sees: one block, all masked
      I.tail_pg = x.lpl < TC_P && x.pg1 - 1 - first < I.n_pg ? x.pg1 - 1 - first : -1;
      I.lpl = x.lpl;
      I.piece = x.base < 0 ? -1 : x.base + sp * x.nt + i0;
      a.items[x.item0 + k] = I;
    }
    if (x.base >= 0) {
      int4* to = x.causal ? a.rest : a.fold;
      for (int k = lane; k < x.nt; k += 32) to[x.t0 + k] = make_int4(x.base + k, x.splits, x.nt, 0);
    } else {  // no pieces: the tiles write these rows
      for (int k = lane; k < x.nt; k += 32) a.rest[x.t0 + k] = make_int4(0, 0, 0, 1);
    }
  }
  __syncthreads();
  const int n_items = room ? item0 : 0;
  // ---- the one-token sequences' list: their pages after the shared ones
  int base_seq = 0, base_pg = 0;
  for (int c0 = 0; c0 < a.n_seqs; c0 += blockDim.x) {
    const int s = c0 + tid;
    int is = 0, np = 0;
    SeqInfo q{};
    if (s < a.n_seqs) {
      q = seq_info(a, s);
      if (q.ok && q.ql == 1) {
        is = 1;
        np = q.pages - a.seq_np[s];
      }
    }
    int tot_seq, tot_pg;
    const int d = base_seq + block_excl_scan(is, warp_sum, &tot_seq);
    const int off = base_pg + block_excl_scan(np, warp_sum, &tot_pg);
    if (is) {
      a.rows[d] = q.q0;
      a.list[d] = make_int2(off, np);
    }
    // the warp writes its sequences' pages one sequence at a time
    for (int l = 0; l < 32; ++l) {
      if (!__shfl_sync(0xffffffffu, is, l)) continue;
      const int dn = __shfl_sync(0xffffffffu, d, l), on = __shfl_sync(0xffffffffu, off, l);
      const int nn = __shfl_sync(0xffffffffu, np, l), lp = __shfl_sync(0xffffffffu, q.lpl, l);
      const int from = __shfl_sync(0xffffffffu, q.pa + q.pages - np, l);
      for (int p = lane; p < nn && int64_t(on) + nn <= a.total_pages; p += 32) {
        int id = a.kv_indices[from + p];
        if (id < 0 || id >= a.num_blocks) {
          flag(a.st, PKV_DEV_SLOT_OOB);
          id = -1;  // no keys
        }
        const int first = p == 0, last = p == nn - 1;
        a.desc[on + p] = make_int2(id, (dn << 7) | (first << 6) | (last << 5) | (last ? lp : TC_P));
      }
    }
    base_seq += tot_seq;
    base_pg += tot_pg;
  }
  // overlapping page lists (some indptr entry runs backwards) list more pages
  // than there are: nothing is streamed
  const bool over = base_pg > a.total_pages;
  const int P = over ? 0 : base_pg;
  // CTAs that stream first: all when there are no tiles, else those that the tiles'
  // one round leaves, stream_least to 7/4 an SM. 32 groups of 8 sequences (the
  // streaming's time is 9 of the tiles'): 1, 5/4, 3/2, 7/4, 2 an SM 58.0, 54.0,
  // 50.8, 49.4, 50.5 us; 256 sequences on a 4096-token prefix (2 of the tiles', 256
  // items): 48.5, 44.5, 58.1, 59.0, 58.5, as left by the round (188 of 444 CTAs) 43.9.
  const int most_stream = a.sms * 7 / 4;
  int n_stream = P == 0       ? 0
                 : n_items == 0 ? a.grid
                                : int(max(int64_t(n_lo), min(int64_t(most_stream), a.grid - int64_t(n_items) * a.n_kv)));
  n_stream = min(n_stream, (P * a.n_kv + SH_WARPS - 1) / SH_WARPS);
  const int ranges = P == 0 ? 0 : max(1, min(P, n_stream * SH_WARPS / a.n_kv));
  __syncthreads();
  for (int d = tid; d < base_seq; d += blockDim.x) {
    const int2 r = a.list[d];
    // ranges [r P / ranges, (r + 1) P / ranges) that hold its pages; (range, sequence) is piece range + d
    const int r0 = P ? int((int64_t(r.x + 1) * ranges + P - 1) / P) - 1 : 0;
    const int r1 = P ? int((int64_t(r.x + r.y) * ranges + P - 1) / P) - 1 : -1;
    a.rest[a.rows[d]] = make_int4(int(a.pieces_cap) + d + r0, r1 - r0 + 1, 1, 0);
  }
  if (tid == 0) {
    if (!room) flag(a.st, PKV_DEV_WORKSPACE);
    if (over) flag(a.st, PKV_DEV_META_BAD);
    a.ctl->n_items = n_items;
    a.ctl->n_stream = n_stream;
    a.ctl->n_ranges = ranges;
    a.ctl->listed = P;
  }
  // read by later kernels before their griddepcontrol.wait (this kernel never
  // triggers its dependents early): visible at GPU scope before the block exits
  __threadfence();
}

// ---------------------------------------------------------------- roles
struct ShArgs {
  const void* q;
  void* out;
  const ShCtl* ctl;
  int32_t* claim;
  const ShItem* items;
  const int2* desc;
  const int32_t* rows;
  const int32_t* kv_indices;
  const char* k_slab;
  const char* v_slab;
  float* part_o;
  float2* part_ml;
  int32_t* st;
  int64_t num_blocks;
  int stream_piece0;  // first piece row of the streaming warps
  int n_heads, n_kv, layer, n_tokens, n_seqs;
  float scale_log2;
};

// Stream role, one warp: KV head h over the listed pages [p0, p1) (range `r`).
// Each sequence it meets leaves the piece (O / l, m, l) of its pages in the
// range. Pages come through the warp's ring of SH_SST stages (cp.async, 128-byte
// rows swizzled for ldmatrix); S^T = K q^T and O^T += V^T P^T on 16-key tiles with
// fp32 online softmax; keys past a page's tokens are neither read nor counted.
template <typename T, int G>
__device__ __forceinline__ void stream_range(const ShArgs& a, unsigned char* ring, int h, int r, int p0, int p1,
                                             int2 cur, int2 nxt, int lane) {
  const int g = lane >> 2, c4 = lane & 3;
  const T* q = static_cast<const T*>(a.q);
  const int n = p1 - p0;
  const uint32_t ring0 = smem_u32(ring);
  const int64_t row_b = int64_t(a.n_kv) * TC_D * 2;
  const int r0 = lane >> 3, ch = lane & 7;  // this lane's chunk of the rows r0, r0 + 4, ... it copies
  const int64_t lane_off = int64_t(r0) * row_b + int64_t(h) * TC_D * 2 + ch * 16;
  // descriptors: lane j holds pages wb + j (cur) and wb + 32 + j (nxt)
  int wb = 0;
  auto desc_at = [&](int i) -> int2 {  // uniform i in [wb, wb + 64)
    const bool in_cur = i < wb + 32;
    return make_int2(__shfl_sync(0xffffffffu, in_cur ? cur.x : nxt.x, i & 31),
                     __shfl_sync(0xffffffffu, in_cur ? cur.y : nxt.y, i & 31));
  };
  auto slide_to = [&](int i) {  // make [i, i + 32) resident
    if (i >= wb + 32) {
      wb += 32;
      cur = nxt;
      nxt = wb + 32 + lane < n ? __ldcg(a.desc + p0 + wb + 32 + lane) : make_int2(-1, 0);
    }
  };
  auto load = [&](int i) {  // page i of the range
    const int2 d = desc_at(i);
    const int valid = d.x < 0 ? 0 : d.y & 31;
    const uint32_t dst = ring0 + (i % SH_SST) * SH_STAGE;
    const int64_t off0 = int64_t(d.x) * TC_P * row_b + lane_off;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int rr = 4 * c + r0;
      const bool ok = rr < valid;
      const int64_t off = ok ? off0 + 4 * c * row_b : 0;
      const uint32_t sw = rr * 128 + ((ch ^ (rr & 7)) << 4);
      cp_async16(dst + sw, a.k_slab + off, ok);
      cp_async16(dst + SH_TILE + sw, a.v_slab + off, ok);
    }
  };
  // B operand of list entry sq's queries of this KV head (plain loads: the
  // kernel that writes them may still run when this one starts)
  auto load_q = [&](int sq, uint32_t (&qb)[4][2]) {
    const int row = sq < a.n_seqs ? __ldcg(a.rows + sq) : -1;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) qb[ks][0] = qb[ks][1] = 0u;
    if (g < G && row >= 0 && row < a.n_tokens) {
      const T* qr = q + (int64_t(row) * a.n_heads + h * G + g) * TC_D + 2 * c4;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        qb[ks][0] = *reinterpret_cast<const uint32_t*>(qr + ks * 16);
        qb[ks][1] = *reinterpret_cast<const uint32_t*>(qr + ks * 16 + 8);
      }
    }
  };
  const int k_tok = lane & 15, k_chk = lane >> 4;
  const int v_tok = (lane & 7) + ((lane >> 4) << 3), v_chk = (lane >> 3) & 1;
#pragma unroll
  for (int i = 0; i < SH_SST - 1; ++i) {
    if (i < n) load(i);
    cp_async_commit();
  }
  int sq = desc_at(0).y >> 7;
  const int sq_last = __ldcg(&a.desc[p1 - 1].y) >> 7;
  uint32_t qb[4][2];
  load_q(sq, qb);
  float o[4][4];
  float m0 = -1e30f, m1 = -1e30f, l0 = 0.f, l1 = 0.f;
#pragma unroll
  for (int mt = 0; mt < 4; ++mt)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[mt][e] = 0.f;
  for (int i = 0; i < n; ++i) {
    slide_to(i);
    if (i + SH_SST - 1 < n) load(i + SH_SST - 1);
    cp_async_commit();
    cp_async_wait<SH_SST - 1>();
    __syncwarp();
    const int2 d = desc_at(i);
    const int valid = d.x < 0 ? 0 : d.y & 31;
    const uint32_t src = ring0 + (i % SH_SST) * SH_STAGE;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      uint32_t af[4];
      const int chunk = 2 * ks + k_chk;
      ldsm_x4(af[0], af[1], af[2], af[3], src + k_tok * 128 + ((chunk ^ (k_tok & 7)) << 4));
      MmaOp<T>::run(s, af, qb[ks][0], qb[ks][1]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] *= a.scale_log2;
    if (valid < TC_P) {
      if (g >= valid) s[0] = s[1] = -INFINITY;
      if (g + 8 >= valid) s[2] = s[3] = -INFINITY;
    }
    float x0 = fmaxf(s[0], s[2]), x1 = fmaxf(s[1], s[3]);
    if (__any_sync(0xffffffffu, x0 > m0 + TC_RESCALE || x1 > m1 + TC_RESCALE)) {
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, off));
        x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, off));
      }
      const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
      const float al0 = ex2(m0 - n0), al1 = ex2(m1 - n1);
      m0 = n0;
      m1 = n1;
      l0 *= al0;
      l1 *= al1;
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        o[mt][0] *= al0;
        o[mt][2] *= al0;
        o[mt][1] *= al1;
        o[mt][3] *= al1;
      }
    }
    const float p00 = ex2(s[0] - m0), p01 = ex2(s[1] - m1);
    const float p10 = ex2(s[2] - m0), p11 = ex2(s[3] - m1);
    l0 += p00 + p10;
    l1 += p01 + p11;
    // P in the pool dtype, the product's operand type (see tl_exp64_smem)
    const uint32_t pb0 = movmatrix_t(MmaOp<T>::pack(p00, p01)), pb1 = movmatrix_t(MmaOp<T>::pack(p10, p11));
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
      uint32_t af[4];
      const int chunk = 2 * mt + v_chk;
      ldsm_x4_t(af[0], af[1], af[2], af[3], src + SH_TILE + v_tok * 128 + ((chunk ^ (v_tok & 7)) << 4));
      MmaOp<T>::run(o[mt], af, pb0, pb1);
    }
    if (((d.y >> 5) & 1) || i == n - 1) {
      // the sequence's last page of the range: its piece, then the next sequence's queries
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, off);
        l1 += __shfl_xor_sync(0xffffffffu, l1, off);
      }
      const float i0 = l0 > 0.f ? 1.f / l0 : 0.f, i1 = l1 > 0.f ? 1.f / l1 : 0.f;
      const int64_t e = int64_t(a.stream_piece0 + r + sq) * a.n_heads + h * G;
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        if (2 * c4 < G) {
          float* po = a.part_o + (e + 2 * c4) * TC_D + mt * 16 + g;
          __stcg(po, o[mt][0] * i0);
          __stcg(po + 8, o[mt][2] * i0);
        }
        if (2 * c4 + 1 < G) {
          float* po = a.part_o + (e + 2 * c4 + 1) * TC_D + mt * 16 + g;
          __stcg(po, o[mt][1] * i1);
          __stcg(po + 8, o[mt][3] * i1);
        }
      }
      if (g == 0) {
        if (2 * c4 < G) __stcg(a.part_ml + e + 2 * c4, make_float2(m0, l0));
        if (2 * c4 + 1 < G) __stcg(a.part_ml + e + 2 * c4 + 1, make_float2(m1, l1));
      }
      ++sq;
      if (sq <= sq_last) load_q(sq, qb);
      m0 = m1 = -1e30f;
      l0 = l1 = 0.f;
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[mt][x] = 0.f;
    }
    __syncwarp();  // every lane has read the stage before its slot is filled again
  }
  cp_async_wait<0>();
}

// O row *= alpha (the lazy rescale). In line, 16 columns at a time after the
// block's scores are dead: 16 registers, no call and none of a call's saves. With
// the epilogue's two halves it took the kernel's local memory from 56 to 24 bytes
// a thread (8 query heads a KV head) and 24 sequences of up to 12 new tokens over
// 2048 shared ones from 18.4 to 17.1 us.
__device__ __forceinline__ void sh_rescale_o(uint32_t tO, float alpha) {
#pragma unroll 1
  for (int q = 0; q < 4; ++q) {
    uint32_t o[16];
    tmem_ld16(tO + q * 16, o);
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
    tmem_st16(tO + q * 16, o);
  }
}

// Tile role: the pipeline of prefill_tc_lean_kernel (pkv_prefill_tc.cu) over the
// plan's items: warp 0 claims items and loads the query tile and the K / V blocks
// by TMA, warp 1 issues S = Q K^T and O += P V (tcgen05, accumulators in TMEM),
// warps 2-5 hold one row a thread: running maximum and sum, P to shared memory,
// lazy rescale of O. The epilogue writes the row as a piece: O / l in fp32 and
// (m, l). The first item of the CTAs that start with tiles is their own number.
//
// What bounds it: a block's chain takes a CTA 1800 cycles (clock64 in a warp: its
// 64 exponentials 770, the maximum 300, the scores from tensor memory 85, the proxy
// fence 100, the rest three barrier turns), three CTAs overlap to 860 a block and
// SM, of which the exponential unit's share is 512; an item's epilogue 3000. From
// launch to the first scores 2 us. 256 sequences on 8192 shared tokens (32 heads, 8
// KV heads: 17 GFLOP in tiles): 46 us with the merge.
template <typename T, int G>
__global__ void __launch_bounds__(TC_THREADS, SH_MINB) shared_kernel(
    const __grid_constant__ CUtensorMap tmap, const __grid_constant__ CUtensorMap qmap, const ShArgs a) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ int s_first;
  __shared__ uint32_t s_tmem;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // ---- tensor memory: 128 columns S | O, freed on every path below. Allocated
  // first thing by every CTA, streaming ones too: the next CTA of the launch
  // starts on an SM only once the one before has given up its allocation permit
  // (measured: a CTA that kept it held the SM at two CTAs until it ended). It is
  // held while the kernels before this one end, and they need none of it: each
  // kernel that allocates lets its successor start only after it has.
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)),
                 "r"(SH_TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    pdl_trigger();  // after the allocation: the next kernel's may follow
  }
  // frees the tensor memory; all threads, after every role is done with it
  auto leave = [&]() {
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
      tc_fence_after();
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(s_tmem), "r"(SH_TMEM_COLS) : "memory");
    }
    if (threadIdx.x == 0) tl_count_exit(a.claim);
  };
  // the plan completed before this kernel could start and fenced its stores
  const int n_items = __ldcg(&a.ctl->n_items) * a.n_kv;
  const int n_stream = __ldcg(&a.ctl->n_stream);
  const int n_tile = int(gridDim.x) - n_stream;  // CTAs [0, n_tile) start with tiles
  const bool streams = int(blockIdx.x) >= n_tile;
  if (!streams && int(blockIdx.x) >= n_items) {  // nothing for this CTA (uniform over the CTA)
    pdl_wait();                                  // the counters belong to the previous launch until it completed
    leave();
    return;
  }
  if (streams) {
    const int ranges = __ldcg(&a.ctl->n_ranges), P = __ldcg(&a.ctl->listed);
    const int w = (int(blockIdx.x) - n_tile) * SH_WARPS + warp;
    bool waited = false;
    for (int u = w; u < ranges * a.n_kv; u += n_stream * SH_WARPS) {
      const int h = u % a.n_kv, r = u / a.n_kv;
      const int p0 = int(int64_t(r) * P / ranges), p1 = int(int64_t(r + 1) * P / ranges);
      // the range's first page descriptors (the plan's: read ahead of the wait)
      const int2 cur = lane < p1 - p0 ? __ldcg(a.desc + p0 + lane) : make_int2(-1, 0);
      const int2 nxt = 32 + lane < p1 - p0 ? __ldcg(a.desc + p0 + 32 + lane) : make_int2(-1, 0);
      if (!waited) pdl_wait();  // q and this layer's appended K/V rows are written by earlier kernels
      waited = true;
      stream_range<T, G>(a, smem_raw + size_t(warp) * SH_SST * SH_STAGE, h, r, p0, p1, cur, nxt, lane);
    }
    if (!waited) pdl_wait();
    // the ring's generic-proxy accesses before the tiles' TMA writes
    fence_proxy_async_smem();
    if (threadIdx.x == 0) s_first = n_tile < n_items ? n_tile + atomicAdd(a.claim, 1) : n_items;
    __syncthreads();
    if (s_first >= n_items) {
      leave();
      return;
    }
  } else if (threadIdx.x == 0) {
    s_first = blockIdx.x;
  }
  // 1024-byte aligned by its declaration: every address below is a constant
  unsigned char* smem = smem_raw;
  unsigned char* qbuf = smem;                             // [128 rows][128 B], 128B swizzle
  unsigned char* kst = smem + TC_QTILE;                   // SH_KST x K [64 keys][128 B]
  unsigned char* vst = kst + size_t(SH_KST) * TC_KTILE;   // SH_VST x V [64 keys][128 B]
  unsigned char* pbuf = vst + size_t(SH_VST) * TC_KTILE;  // P [128 rows][128 B], 128B swizzle
  uint64_t* kfull = reinterpret_cast<uint64_t*>(pbuf + TC_QTILE);
  uint64_t* kempty = kfull + SH_KST;
  uint64_t* vfull = kempty + SH_KST;
  uint64_t* vempty = vfull + SH_VST;
  uint64_t* s_full = vempty + SH_VST;
  uint64_t* s_free = s_full + 1;
  uint64_t* p_full = s_free + 1;
  uint64_t* pv_done = p_full + 1;
  uint64_t* q_full = pv_done + 1;
  uint64_t* q_empty = q_full + 1;
  uint64_t* o_free = q_empty + 1;
  uint64_t* item_full = o_free + 1;
  uint64_t* item_empty = item_full + 2;
  uint64_t* drain = item_empty + 2;
  __shared__ ShItem s_item[2];

  if (threadIdx.x == 0) {
    prefetch_tmap(&tmap);
    prefetch_tmap(&qmap);
    for (int i = 0; i < SH_KST; ++i) {
      mbar_init(&kfull[i], 1);
      mbar_init(&kempty[i], 1);
    }
    for (int i = 0; i < SH_VST; ++i) {
      mbar_init(&vfull[i], 1);
      mbar_init(&vempty[i], 1);
    }
    mbar_init(s_full, 1);
    mbar_init(s_free, 4);
    mbar_init(p_full, 4);
    mbar_init(pv_done, 1);
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    mbar_init(o_free, 4);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], 5);
    }
    mbar_init(drain, 1);
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = s_tmem;
  const uint32_t tO = tbase + TC_KB;
  // The kernels before this one may run for as long as they need: the bounded
  // waits below count from their completion (warp 0 waits once it has read the
  // plan's part of its first item).
  if (warp != 0) pdl_wait();

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    const int kvc = 2 * a.layer;
    uint32_t kiss = 0, viss = 0, qiss = 0;  // K / V slots and query tiles filled so far
    int it = 0;                   // items published
    bool dead = false;
    int w = s_first;
    while (!dead) {
      const bool end = w >= n_items;
      ShItem I{};
      if (!end) {
        const int4* d = reinterpret_cast<const int4*>(a.items + w / a.n_kv);
        const int4 x = __ldg(d), y = __ldg(d + 1), z = __ldg(d + 2);
        I = ShItem{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w, z.x, z.y, w % a.n_kv, 0};
      }
      const int pg_at = I.pg_at;
      bool pg_bad = false;
      for (int pg = lane; pg < I.n_pg; pg += 32) {
        const int id = a.kv_indices[pg_at + pg];
        pg_bad |= id < 0 || id >= a.num_blocks;
      }
      pg_bad = __any_sync(0xffffffffu, pg_bad);
      // q, this layer's appended K/V rows and the pieces' last readers: the first
      // item is the plan's and was read ahead of the wait
      if (it == 0) pdl_wait();
      const int sl = it & 1;
      if (it >= 2 && !mbar_wait_bounded_sleepy(&item_empty[sl], ((it - 2) >> 1) & 1, a.st, 32)) dead = true;
      dead = __any_sync(0xffffffffu, dead);
      if (dead) break;
      if (lane == 0) {
        I.zero = pg_bad ? 1 : 0;
        if (end) I.nblk = 0;
        s_item[sl] = I;
        if (pg_bad) flag(a.st, PKV_DEV_SLOT_OOB);
        mbar_arrive(&item_full[sl]);
      }
      __syncwarp();
      if (end) break;
      if (lane == 0) {
        // four pages' rows of block j; a page past the range reads the zero fill of a negative coordinate
        auto load = [&](unsigned char* dst, uint64_t* full, int j, int kv) {
          mbar_arrive_expect_tx(full, TC_KTILE);
#pragma unroll
          for (int u = 0; u < TC_PPB; ++u) {
            const int pg = j * TC_PPB + u;
            const int row = pg < I.n_pg && !pg_bad ? a.kv_indices[pg_at + pg] * TC_P : -TC_P;
            tma_load_4d(dst + u * TC_PAGE, &tmap, full, 0, row, I.h, kv);
          }
        };
        auto load_k = [&](int j) {
          const int st = int(kiss % SH_KST);
          if (kiss >= SH_KST && !mbar_wait_bounded_sleepy(&kempty[st], ((kiss / SH_KST) - 1) & 1, a.st, 32)) {
            dead = true;
            return;
          }
          load(kst + size_t(st) * TC_KTILE, &kfull[st], j, kvc);
          ++kiss;
        };
        // the query tile: first thing, or once the item before has read its own
        if (it >= 1) {
          for (int j = 0; j < SH_KST - 1 && j < I.nblk && !dead; ++j) load_k(j);
          if (!dead && !mbar_wait_bounded_sleepy(q_empty, (it - 1) & 1, a.st, 64)) dead = true;
        }
        if (!dead) {
          mbar_arrive_expect_tx(q_full, TC_QTILE);
          tma_load_3d(qbuf, &qmap, q_full, 0, I.h * G, I.t0);
          ++qiss;
        }
        if (it == 0)
          for (int j = 0; j < SH_KST - 1 && j < I.nblk && !dead; ++j) load_k(j);
        for (int j = 0; j < I.nblk && !dead; ++j) {
          if (j + SH_KST - 1 < I.nblk) load_k(j + SH_KST - 1);
          if (dead) break;
          // the next item, two blocks before it is needed. No claim where the CTAs' own
          // numbers cover the items: atomics on one address take turns
          if (j == I.nblk - 1) w = n_tile < n_items ? n_tile + atomicAdd(a.claim, 1) : n_items;
          const int st = int(viss % SH_VST);
          if (viss >= SH_VST && !mbar_wait_bounded_sleepy(&vempty[st], ((viss / SH_VST) - 1) & 1, a.st, 32)) {
            dead = true;
            break;
          }
          load(vst + size_t(st) * TC_KTILE, &vfull[st], j, kvc + 1);
          ++viss;
        }
      }
      dead = __shfl_sync(0xffffffffu, dead, 0);
      ++it;
      w = __shfl_sync(0xffffffffu, w, 0);
    }
    if (dead && lane == 0) {
      // let this CTA's own copies land before its shared memory can be released
      for (uint32_t i = kiss > SH_KST ? kiss - SH_KST : 0; i < kiss; ++i)
        mbar_wait_bounded(&kfull[i % SH_KST], (i / SH_KST) & 1, nullptr);
      for (uint32_t i = viss > SH_VST ? viss - SH_VST : 0; i < viss; ++i)
        mbar_wait_bounded(&vfull[i % SH_VST], (i / SH_VST) & 1, nullptr);
      if (qiss >= 1) mbar_wait_bounded(q_full, (qiss - 1) & 1, nullptr);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    constexpr int fmt = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
    constexpr uint32_t idS = idesc_f16(fmt, 0, TC_KB);
    constexpr uint32_t idPV = idesc_f16(fmt, 1, TC_D);
    const uint32_t q_addr = smem_u32(qbuf), p_addr = smem_u32(pbuf);
    uint32_t g = 0;
    int it = 0;
    bool dead = false;
    auto pv = [&](uint32_t gp, int jp, const ShItem& I) -> bool {
      const int stp = int(gp % SH_VST);
      bool bad = !mbar_wait_bounded(p_full, gp & 1, a.st);
      if (!bad && jp == 0 && it >= 1 && !mbar_wait_bounded(o_free, (it - 1) & 1, a.st)) bad = true;
      if (!bad && !mbar_wait_bounded(&vfull[stp], (gp / SH_VST) & 1, a.st)) bad = true;
      bad = __any_sync(0xffffffffu, bad);
      if (bad) return false;
      if (I.tail_pg >= 0 && jp == I.tail_pg / TC_PPB) {
        // rows lpl..15 of the last page's V slice were never written: zero them
        uint4* vt = reinterpret_cast<uint4*>(vst + size_t(stp) * TC_KTILE + (I.tail_pg - jp * TC_PPB) * TC_PAGE);
        for (int rr = I.lpl * 8 + lane; rr < TC_P * 8; rr += 32) vt[rr] = make_uint4(0u, 0u, 0u, 0u);
        fence_proxy_async_smem();
        __syncwarp();
      }
      if (lane == 0) {
        tc_fence_after();
        const uint32_t vaddr = smem_u32(vst + size_t(stp) * TC_KTILE);
#pragma unroll
        for (int kk = 0; kk < TC_KB / 16; ++kk)
          umma_ss(tO, sw128_desc(p_addr + 32 * kk), sw128_desc(vaddr + 16 * 128 * kk), idPV,
                  (jp > 0 || kk > 0) ? 1u : 0u);
        umma_commit(&vempty[stp]);
        umma_commit(pv_done);
      }
      __syncwarp();
      return true;
    };
    while (!dead) {
      const int sl = it & 1;
      if (!mbar_wait_bounded(&item_full[sl], (it >> 1) & 1, a.st)) dead = true;
      dead = __any_sync(0xffffffffu, dead);
      if (dead) break;
      const ShItem I = s_item[sl];
      if (I.nblk == 0) break;
      if (!mbar_wait_bounded(q_full, it & 1, a.st)) dead = true;
      dead = __any_sync(0xffffffffu, dead);
      if (dead) break;
      for (int j = 0; j < I.nblk; ++j) {
        const uint32_t gj = g + j;
        const int st = int(gj % SH_KST);
        // S_j overwrites S_{j-1}: after the softmax threads loaded it
        if (gj >= 1 && !mbar_wait_bounded(s_free, (gj - 1) & 1, a.st)) dead = true;
        if (!dead && !mbar_wait_bounded(&kfull[st], (gj / SH_KST) & 1, a.st)) dead = true;
        dead = __any_sync(0xffffffffu, dead);
        if (dead) break;
        if (lane == 0) {
          tc_fence_after();
          const uint32_t kaddr = smem_u32(kst + size_t(st) * TC_KTILE);
#pragma unroll
          for (int kk = 0; kk < TC_D / 16; ++kk)
            umma_ss(tbase, sw128_desc(q_addr + 32 * kk), sw128_desc(kaddr + 32 * kk), idS, kk > 0);
          umma_commit(s_full);
          umma_commit(&kempty[st]);
          if (j == I.nblk - 1) umma_commit(q_empty);  // the item's last read of its query tile
        }
        __syncwarp();
        if (j >= 1 && !pv(gj - 1, j - 1, I)) {
          dead = true;
          break;
        }
      }
      if (dead) break;
      if (!pv(g + I.nblk - 1, I.nblk - 1, I)) {
        dead = true;
        break;
      }
      if (lane == 0) mbar_arrive(&item_empty[sl]);
      g += I.nblk;
      ++it;
    }
    // every MMA issued above has completed before TMEM is freed
    if (lane == 0) {
      umma_commit(drain);
      mbar_wait_bounded(drain, 0, a.st);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ softmax warps
    const int q4 = warp & 3;       // TMEM lane quarter this warp may access
    const int r = q4 * 32 + lane;  // this thread's row: token r / G, query head r % G of the item's group
    const uint32_t lane_off = uint32_t(q4 * 32) << 16;
    const float sl2 = a.scale_log2;
    const float sc = sl2 > 0.f ? sl2 : 1.f;  // the scale still to apply after masking (log2 units)
    unsigned char* prow = pbuf + r * 128;
    uint32_t g = 0;
    int it = 0;
    bool dead = false;
    while (!dead) {
      const int sl = it & 1;
      if (!mbar_wait_bounded(&item_full[sl], (it >> 1) & 1, a.st)) dead = true;
      dead = __any_sync(0xffffffffu, dead);
      if (dead) break;
      const int nblk = s_item[sl].nblk;
      if (nblk == 0) break;
      const int nt = s_item[sl].nt;
      // last key of the range this row sees. A row past the tile's tokens is not
      // masked (the mask costs its warp 550 of 2400 cycles a block): nothing reads it
      const int lim = r / G < nt ? s_item[sl].lim0 + s_item[sl].causal * (r / G) : 0x7fffffff;
      // no token in this warp's 32 rows: only the barriers. Its rows of P hold
      // anything: they reach its own rows of O alone, which nothing reads
      const bool idle = q4 * 32 / G >= nt;
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < nblk; ++j) {
        const uint32_t gj = g + j;
        if (!mbar_wait_bounded(s_full, gj & 1, a.st)) dead = true;
        dead = __any_sync(0xffffffffu, dead);
        if (dead) break;
        tc_fence_after();
        if (idle) {
          if (lane == 0) mbar_arrive(s_free);
          if (gj >= 1 && !mbar_wait_bounded(pv_done, (gj - 1) & 1, a.st)) dead = true;
          dead = __any_sync(0xffffffffu, dead);
          if (dead) break;
          if (lane == 0) mbar_arrive(p_full);
          continue;
        }
        uint32_t sr[64];
        tmem_ld64(tbase + lane_off, sr);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_free);  // S_{j+1} may overwrite S now
        const int kb0 = j * TC_KB;
        if (sl2 <= 0.f) {  // a non-positive scale: scale first so the masked -inf stays the minimum
#pragma unroll
          for (int i = 0; i < 64; ++i) sr[i] = __float_as_uint(__uint_as_float(sr[i]) * sl2);
        }
        if (kb0 + TC_KB - 1 > lim) {  // the block reaches past this row's last visible key
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (kb0 + i > lim) sr[i] = __float_as_uint(-INFINITY);
        }
        float mx;
        {
          float t[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) t[u] = __uint_as_float(sr[u]);
#pragma unroll
          for (int i = 8; i < 64; i += 2)
            t[(i >> 1) & 7] = max3f(t[(i >> 1) & 7], __uint_as_float(sr[i]), __uint_as_float(sr[i + 1]));
          mx = max3f(max3f(t[0], t[1], t[2]), max3f(t[3], t[4], t[5]), fmaxf(t[6], t[7]));
        }
        mx = mx * sc;  // -inf stays -inf (sc > 0)
        const float mn = fmaxf(m, mx);
        float m_new = m;
        if (mn != -INFINITY && (m == -INFINITY || mn > m + TC_RESCALE)) m_new = mn;
        const bool resc = (m_new != m) && (m != -INFINITY);  // earlier blocks already added to O
        const float alpha = resc ? ex2(m - m_new) : 1.f;
        l *= alpha;
        m = m_new;
        // P.V_{j-1} done: the P tile is free and O holds every earlier block
        if (gj >= 1 && !mbar_wait_bounded(pv_done, (gj - 1) & 1, a.st)) dead = true;
        dead = __any_sync(0xffffffffu, dead);
        if (dead) break;
        const float mu = m == -INFINITY ? 0.f : m;
        tl_exp64_smem<T>(sr, f32x2(sc, sc), f32x2(-mu, -mu), l, prow, r);
        fence_proxy_async_smem();  // P (generic-proxy stores) -> the P.V MMA (async proxy)
        if (__any_sync(0xffffffffu, resc)) {
          tc_fence_after();
          sh_rescale_o(tO + lane_off, alpha);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full);
      }
      if (dead) break;
      if (idle) {
        if (lane == 0) {
          mbar_arrive(o_free);
          mbar_arrive(&item_empty[sl]);
        }
        g += nblk;
        ++it;
        continue;
      }
      // ---- epilogue: O / l of the item -> its piece rows in fp32 (or out in the
      // pool dtype), staged through this warp's own rows of the P tile (the
      // item's last P.V completed) 32 columns at a time, so that the stores are
      // whole 128-byte lines
      const uint32_t gl = g + nblk - 1;
      if (!mbar_wait_bounded(pv_done, gl & 1, a.st)) dead = true;
      dead = __any_sync(0xffffffffu, dead);
      if (dead) break;
      tc_fence_after();
      const int h = s_item[sl].h, t0 = s_item[sl].t0, piece = s_item[sl].piece;
      const bool zero = s_item[sl].zero != 0;
      const float inv = (l == 0.f || zero) ? 0.f : 1.f / l;  // rows that saw nothing, or a bad page: zeros (not a NaN sum)
      if (piece >= 0 && r / G < nt)
        __stcg(a.part_ml + int64_t(piece + r / G) * a.n_heads + h * G + r % G,
               make_float2(m == -INFINITY || zero ? -1e30f : m, zero ? 0.f : l));
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        uint32_t o[32];
        tmem_ld32(tO + lane_off + half * 32, o);
        tc_fence_before();
        if (half == 1) {
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(o_free);           // O read: the next item's first P.V may overwrite it
            mbar_arrive(&item_empty[sl]);  // and the item's fields
          }
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(inv == 0.f ? 0.f : __uint_as_float(o[i]) * inv);
        if (piece >= 0) {
#pragma unroll
          for (int c = 0; c < 8; ++c)
            *reinterpret_cast<uint4*>(prow + ((c ^ (r & 7)) << 4)) =
                make_uint4(o[c * 4], o[c * 4 + 1], o[c * 4 + 2], o[c * 4 + 3]);
          __syncwarp();
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) {
            const int rw = q4 * 32 + 4 * kk + (lane >> 3);
            const uint4 v = *reinterpret_cast<const uint4*>(pbuf + rw * 128 + (((lane & 7) ^ (rw & 7)) << 4));
            if (rw / G < nt)
              __stcg(reinterpret_cast<uint4*>(a.part_o + (int64_t(piece + rw / G) * a.n_heads + h * G + rw % G) * TC_D +
                                              half * 32) + (lane & 7), v);
          }
        } else {  // 32 columns in the pool dtype: half a line a row
          T* out = static_cast<T*>(a.out);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              w[e] = MmaOp<T>::pack(__uint_as_float(o[c * 8 + 2 * e]), __uint_as_float(o[c * 8 + 2 * e + 1]));
            *reinterpret_cast<uint4*>(prow + ((c ^ (r & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
          }
          __syncwarp();
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const int rw = q4 * 32 + 8 * kk + (lane >> 2);
            const uint4 v = *reinterpret_cast<const uint4*>(pbuf + rw * 128 + (((lane & 3) ^ (rw & 7)) << 4));
            if (rw / G < nt)
              reinterpret_cast<uint4*>(out + (int64_t(t0 + rw / G) * a.n_heads + h * G + rw % G) * TC_D +
                                       half * 32)[lane & 3] = v;
          }
        }
        __syncwarp();  // the staged rows are read: the next half's, or the next P rows, may follow
      }
      g += nblk;
      ++it;
    }
  }

  leave();
}

// the tile role's buffers, or the streaming warps' rings
size_t sh_smem() { return std::max(2 * size_t(TC_QTILE) + size_t(SH_KST + SH_VST) * TC_KTILE + 256, SH_RING); }

// ---------------------------------------------------------------- merge
// One warp per (token, query head): its pieces over the shared keys and over its
// own -> out. Two dims a lane, eight pieces' loads in flight.
template <typename T>
__global__ void __launch_bounds__(256) shared_merge_kernel(const int4* fold, const int4* rest, const float* part_o,
                                                           const float2* part_ml, void* out, int n_tokens,
                                                           int n_heads) {
  const int64_t w = (int64_t(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  pdl_trigger();
  if (w >= int64_t(n_tokens) * n_heads) {
    pdl_wait();
    return;
  }
  const int t = int(w / n_heads), hh = int(w % n_heads);
  const int4 b = __ldcg(rest + t);  // the plan's: complete before any kernel of the step started
  const int4 f = __ldcg(fold + t);
  pdl_wait();
  uint32_t* row = reinterpret_cast<uint32_t*>(static_cast<T*>(out) + (int64_t(t) * n_heads + hh) * TC_D) + lane;
  if (b.y <= 0) {
    if (b.w == 0) *row = 0u;  // its sequence's tables are inconsistent: zeros
    return;
  }
  const int n = f.y + b.y;
  constexpr int U = 8;
  float M = -1e30f, L = 0.f, y0 = 0.f, y1 = 0.f;
  for (int i0 = 0; i0 < n; i0 += U) {
    float2 ml[U], v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u;
      const int64_t p = i < f.y ? int64_t(f.x) + int64_t(i) * f.z : int64_t(b.x) + int64_t(i - f.y) * b.z;
      ml[u] = i < n ? __ldcg(part_ml + p * n_heads + hh) : make_float2(-1e30f, 0.f);
      v[u] = i < n ? __ldcg(reinterpret_cast<const float2*>(part_o + (p * n_heads + hh) * TC_D) + lane)
                   : make_float2(0.f, 0.f);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float Mn = fmaxf(M, ml[u].x);
      const float c = ex2(M - Mn), k = ml[u].y * ex2(ml[u].x - Mn);
      y0 = y0 * c + k * v[u].x;
      y1 = y1 * c + k * v[u].y;
      L = L * c + k;
      M = Mn;
    }
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  *row = MmaOp<T>::pack(y0 * inv, y1 * inv);
}

// ---------------------------------------------------------------- host
bool shared_geometry(const pkv_pool& p, int n_heads) {
  const int g = n_heads / p.n_kv_heads;
  return (p.dtype == PKV_F16 || p.dtype == PKV_BF16) && p.head_dim == TC_D && p.block_size == TC_P &&
         p.n_kv_heads <= 8 && (g == 1 || g == 2 || g == 4 || g == 8);
}

int check_batch(const pkv_batch* b) {
  if (!b) return fail(PKV_ERR_ARG, "batch descriptor is NULL");
  if (b->n_seqs <= 0) return fail(PKV_ERR_ARG, "batch has no sequences");
  if (b->n_tokens < 0 || b->total_pages < 0 || b->total_pages >= (int64_t(1) << 31) || b->n_seqs >= (1 << 24))
    return fail(PKV_ERR_ARG, "bad batch sizes");
  if (!b->cu_query_lens || !b->kv_indptr || !b->kv_last_page_len || (b->total_pages && !b->kv_indices))
    return fail(PKV_ERR_ARG, "batch CSR pointers must be non-NULL");
  return PKV_OK;
}

int check_shared(const pkv_pool* pool, int32_t n_heads, const pkv_batch* b) {
  if (int rc = check_pool(pool)) return rc;
  if (!b) return fail(PKV_ERR_ARG, "batch descriptor is NULL");
  if (n_heads <= 0 || n_heads % pool->n_kv_heads)
    return fail(PKV_ERR_ARG, "n_heads must be a positive multiple of n_kv_heads");
  if (!shared_geometry(*pool, n_heads))
    return fail(PKV_ERR_UNSUPPORTED, "shared-prefix attention takes fp16 / bf16 pools, head_dim 64, 16-token pages, "
                                     "up to 8 KV heads and 1, 2, 4 or 8 query heads per KV head");
  return check_batch(b);
}

int check_groups(const pkv_batch& b, int32_t n_groups, const int32_t* group_indptr, const int32_t* prefix_pages) {
  if (n_groups <= 0 || n_groups > b.n_seqs)
    return fail(PKV_ERR_ARG, "n_groups must be between 1 and the number of sequences");
  if (!group_indptr || !prefix_pages) return fail(PKV_ERR_ARG, "group_indptr and prefix_pages must be non-NULL");
  return PKV_OK;
}

// The step's part of the plan's arguments: what shared_check_kernel reads.
PlanArgs step_args(const pkv_pool& p, const pkv_batch& b, int32_t n_groups, const int32_t* group_indptr,
                   const int32_t* prefix_pages) {
  PlanArgs a{};
  a.cu_q = b.cu_query_lens;
  a.kv_lens = b.kv_lens;
  a.kv_indptr = b.kv_indptr;
  a.kv_indices = b.kv_indices;
  a.last_page_len = b.kv_last_page_len;
  a.group_indptr = group_indptr;
  a.prefix_pages = prefix_pages;
  a.st = b.dev_status;
  a.num_blocks = p.num_blocks;
  a.total_pages = b.total_pages;
  a.n_seqs = b.n_seqs;
  a.n_tokens = b.n_tokens;
  a.n_groups = n_groups;
  a.page = p.block_size;
  return a;
}

template <typename T, int G>
int launch_shared_t(const CUtensorMap& tm, const CUtensorMap& qm, const ShArgs& a, int grid, cudaStream_t s) {
  static std::mutex mu;
  static std::vector<char> ready;
  int dev = 0;
  PKV_CUDA_RET(cudaGetDevice(&dev));
  {
    std::lock_guard<std::mutex> lock(mu);
    if ((int)ready.size() <= dev) ready.resize(dev + 1, 0);
    if (!ready[dev]) {
      PKV_CUDA_RET(cudaFuncSetAttribute(shared_kernel<T, G>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        int(sh_smem())));
      // three CTAs of ~73 KiB need the whole shared-memory carveout
      PKV_CUDA_RET(cudaFuncSetAttribute(shared_kernel<T, G>, cudaFuncAttributePreferredSharedMemoryCarveout,
                                        int(cudaSharedmemCarveoutMaxShared)));
      ready[dev] = 1;
    }
  }
  PKV_CUDA_RET(launch_kernel(shared_kernel<T, G>, dim3(grid), dim3(TC_THREADS), sh_smem(), s, true, tm, qm, a));
  return PKV_OK;
}

template <typename T>
int launch_shared_g(int groups, const CUtensorMap& tm, const CUtensorMap& qm, const ShArgs& a, int grid,
                    cudaStream_t s) {
  switch (groups) {
    case 1: return launch_shared_t<T, 1>(tm, qm, a, grid, s);
    case 2: return launch_shared_t<T, 2>(tm, qm, a, grid, s);
    case 4: return launch_shared_t<T, 4>(tm, qm, a, grid, s);
    case 8: return launch_shared_t<T, 8>(tm, qm, a, grid, s);
  }
  return fail(PKV_ERR_UNSUPPORTED, "shared-prefix attention: unsupported GQA group size");
}

}  // namespace
}  // namespace pkv

using namespace pkv;

extern "C" size_t pkv_shared_workspace_size(const pkv_pool* pool, int32_t n_heads, int32_t n_seqs, int32_t n_tokens,
                                            int64_t total_pages) {
  if (!pool || pool->n_kv_heads <= 0 || n_heads < pool->n_kv_heads || n_seqs <= 0 || n_tokens < 0 || total_pages < 0 ||
      !shared_geometry(*pool, n_heads))
    return 0;
  return sh_layout(n_heads, pool->n_kv_heads, n_seqs, n_tokens, total_pages).total;
}

extern "C" int pkv_plan_shared(const pkv_pool* pool, int32_t n_heads, const pkv_batch* batch, int32_t n_groups,
                               const int32_t* group_indptr, const int32_t* prefix_pages, void* workspace,
                               size_t workspace_bytes, void* stream) {
  if (int rc = check_shared(pool, n_heads, batch)) return rc;
  if (int rc = check_groups(*batch, n_groups, group_indptr, prefix_pages)) return rc;
  const int groups = n_heads / pool->n_kv_heads;
  const ShLayout w = sh_layout(n_heads, pool->n_kv_heads, batch->n_seqs, batch->n_tokens, batch->total_pages);
  if (!workspace || workspace_bytes < w.total)
    return fail(PKV_ERR_ARG, "workspace too small: need " + std::to_string(w.total) + " bytes");
  if (reinterpret_cast<uintptr_t>(workspace) & 255) return fail(PKV_ERR_ARG, "workspace must be 256-byte aligned");
  char* ws = static_cast<char*>(workspace);
  PlanArgs a = step_args(*pool, *batch, n_groups, group_indptr, prefix_pages);
  a.n_kv = pool->n_kv_heads;
  a.tpt = TC_ROWS / groups;
  a.sms = num_sms();
  a.grid = SH_MINB * num_sms();
  a.splits_cap = split_cap(batch->n_tokens);
  a.pieces_cap = w.pieces;
  a.items_cap = w.items_cap;
  a.ctl = reinterpret_cast<ShCtl*>(ws + w.ctl);
  a.rows = reinterpret_cast<int32_t*>(ws + w.rows);
  a.list = reinterpret_cast<int2*>(ws + w.list);
  a.seq_np = reinterpret_cast<int32_t*>(ws + w.seq_np);
  a.group_bad = reinterpret_cast<int32_t*>(ws + w.group_bad);
  a.ents = reinterpret_cast<ShEnt*>(ws + w.ents);
  a.items = reinterpret_cast<ShItem*>(ws + w.items);
  a.desc = reinterpret_cast<int2*>(ws + w.desc);
  a.fold = reinterpret_cast<int4*>(ws + w.fold);
  a.rest = reinterpret_cast<int4*>(ws + w.rest);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  PKV_CUDA_RET(cudaMemsetAsync(a.group_bad, 0, sizeof(int32_t) * size_t(batch->n_seqs), s));
  shared_check_kernel<<<unsigned(batch->n_seqs), 128, 0, s>>>(a);
  PKV_CUDA_RET(cudaGetLastError());
  shared_plan_kernel<<<1, 1024, 0, s>>>(a);
  PKV_CUDA_RET(cudaGetLastError());
  return PKV_OK;
}

extern "C" int pkv_check_shared(const pkv_pool* pool, const pkv_batch* batch, int32_t n_groups,
                                const int32_t* group_indptr, const int32_t* prefix_pages, void* stream) {
  if (int rc = check_pool(pool)) return rc;
  if (int rc = check_batch(batch)) return rc;
  if (int rc = check_groups(*batch, n_groups, group_indptr, prefix_pages)) return rc;
  shared_check_kernel<<<unsigned(batch->n_seqs), 128, 0, static_cast<cudaStream_t>(stream)>>>(
      step_args(*pool, *batch, n_groups, group_indptr, prefix_pages));
  PKV_CUDA_RET(cudaGetLastError());
  return PKV_OK;
}

extern "C" int pkv_attend_shared_planned(const pkv_pool* pool, int32_t layer, int32_t n_heads, const void* q,
                                         void* out, float scale, const pkv_batch* batch, void* workspace,
                                         size_t workspace_bytes, void* stream) {
  if (int rc = check_shared(pool, n_heads, batch)) return rc;
  const pkv_pool& p = *pool;
  if (layer < 0 || layer >= p.num_layers)
    return fail(PKV_ERR_ARG, "layer_idx " + std::to_string(layer) + " out of range [0, " +
                                 std::to_string(p.num_layers) + ")");
  if (batch->n_tokens == 0) return PKV_OK;
  if (!q || !out) return fail(PKV_ERR_ARG, "q and out must be non-NULL");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15)
    return fail(PKV_ERR_ARG, "q and out must be 16-byte aligned");
  const int groups = n_heads / p.n_kv_heads;
  const ShLayout w = sh_layout(n_heads, pool->n_kv_heads, batch->n_seqs, batch->n_tokens, batch->total_pages);
  if (!workspace || workspace_bytes < w.total)
    return fail(PKV_ERR_ARG, "workspace too small: need " + std::to_string(w.total) + " bytes");
  char* ws = static_cast<char*>(workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  CUtensorMap tm, qm;
  if (int rc = pool_tmap_head(p, &tm)) return rc;
  if (int rc = q_tmap(p.dtype, q, batch->n_tokens, n_heads, groups, &qm)) return rc;
  ShArgs a;
  a.q = q;
  a.out = out;
  a.ctl = reinterpret_cast<const ShCtl*>(ws + w.ctl);
  a.claim = reinterpret_cast<ShCtl*>(ws + w.ctl)->claim;
  a.items = reinterpret_cast<const ShItem*>(ws + w.items);
  a.desc = reinterpret_cast<const int2*>(ws + w.desc);
  a.rows = reinterpret_cast<const int32_t*>(ws + w.rows);
  a.kv_indices = batch->kv_indices;
  a.k_slab = static_cast<const char*>(p.base) + int64_t(2) * layer * slab_bytes(p);
  a.v_slab = a.k_slab + slab_bytes(p);
  a.stream_piece0 = int(w.pieces);
  a.n_tokens = batch->n_tokens;
  a.n_seqs = batch->n_seqs;
  a.part_o = reinterpret_cast<float*>(ws + w.part_o);
  a.part_ml = reinterpret_cast<float2*>(ws + w.part_ml);
  a.st = batch->dev_status;
  a.num_blocks = p.num_blocks;
  a.n_heads = n_heads;
  a.n_kv = p.n_kv_heads;
  a.layer = layer;
  a.scale_log2 = scale * 1.4426950408889634f;
  const int grid = SH_MINB * num_sms();
  int rc = p.dtype == PKV_F16 ? launch_shared_g<__half>(groups, tm, qm, a, grid, s)
                              : launch_shared_g<__nv_bfloat16>(groups, tm, qm, a, grid, s);
  if (rc) return rc;
  const int64_t blocks = (int64_t(batch->n_tokens) * n_heads * 32 + 255) / 256;
  if (blocks >= (int64_t(1) << 31)) return fail(PKV_ERR_ARG, "too many tokens for one call");
  auto kern = p.dtype == PKV_F16 ? shared_merge_kernel<__half> : shared_merge_kernel<__nv_bfloat16>;
  PKV_CUDA_RET(launch_kernel(kern, dim3(unsigned(blocks)), dim3(256), 0, s, true,
                             reinterpret_cast<const int4*>(ws + w.fold), reinterpret_cast<const int4*>(ws + w.rest),
                             static_cast<const float*>(a.part_o), static_cast<const float2*>(a.part_ml), out,
                             batch->n_tokens, n_heads));
  return PKV_OK;
}
