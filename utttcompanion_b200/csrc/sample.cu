// Sampling of one token per row from logits, with temperature, top-k, top-p and
// min-p, from one given uniform number per row (the rules of _sample_next_token,
// model/uttt_model.py:1181-1235, plus top-k and min-p; the random number is an
// input, so a pick is repeatable whatever else is in the batch).
//
// Mathematics.  A row's candidates are its ids below active_limit that are not
// PAD / BOS / UNK and whose logit is neither NaN nor -inf.  With m the largest
// logit, w_i = exp((s_i - m) / T).  Candidates are ordered by (s descending, id
// ascending); top-k keeps the first k, top-p those whose mass before them is at
// most top_p times the mass top-k left, min-p those with w_i >= min_p.  All three
// keep a prefix of that order, so the kept set is one cut element.  The pick is
// the lowest id i with (sum of kept w_j, j <= i) > u * (sum of all kept w_j).
//
// Exactness.  w_i is evaluated in 64 bits (table of 2^(j/32) and a short Taylor
// polynomial: the table-driven method of Tang, ACM TOMS 15, 1989) and rounded
// once to a whole number of 2^-45, so every sum of weights is an exact 64-bit
// integer that does not depend on the order of the additions: histograms with
// atomics, splits over CTAs and any grid give the same cut and the same pick.
// A rounding moves a sum of n weights by at most n * 2^-46 of the largest one.
//
// Layout.  One cluster of S CTAs per row; CTA r keeps its part of the row's
// logits in shared memory as order-preserving 32-bit keys, read from HBM once.
// A cut is found by a histogram over 2048 bins of the exponent (linear in
// s - m), merged over the cluster in distributed shared memory, and the few
// candidates of the bin that holds it are ranked against each other; a bin with
// too many (equal or nearly equal logits) is split again by the bits of its
// (key, id) pairs until few are left.
#include <cooperative_groups.h>

#include "common.cuh"
#include "host_util.cuh"

namespace cg = cooperative_groups;

namespace uttt {
namespace {

constexpr int SM_THREADS = 512;
constexpr int SM_WARPS = SM_THREADS / 32;
constexpr int SM_BINS = 2048;
constexpr int SM_CAP = 256;              // candidates ranked against each other directly
constexpr int SM_MAX_CTAS = 8;
constexpr int SM_MAX_V = 262144;         // 8 CTAs of 32768 keys
constexpr double SM_RANGE = 46.0;        // weights below 2^-46 round to zero
constexpr float SM_GREEDY_T = 1e-5f;     // _sample_next_token's greedy border

typedef unsigned long long u64;

struct Sel {     // value exchanged between the CTAs of a cluster
  u64 a, b;
};

struct SampleShared {
  double tab[32];                        // 2^(j / 32)
  Sel xch[2][SM_MAX_CTAS];               // one slot per CTA, two phases
  u64 wred[SM_WARPS], wred2[SM_WARPS];
  u64 cand[2][SM_CAP];                   // rank 0: gathered candidates; others: their copies of them
  u64 cand_w[SM_CAP];
  unsigned n_cand[2];                    // rank 0; gathers alternate between the two lists
  u64 res_base, res_cut;
  int res_bin;
  unsigned hist[3][SM_BINS];             // count, or 16-bit limbs of the mass
};

// order-preserving key of a logit: larger logit, larger key; 0 for excluded ones.  Both zeros are one value.
__device__ __forceinline__ unsigned order_key(unsigned bits) {
  if ((bits << 1) > 0xff000000u || bits == 0xff800000u) return 0u;   // NaN, -inf
  if ((bits << 1) == 0u) bits = 0u;
  return (bits & 0x80000000u) ? ~bits : (bits | 0x80000000u);
}
__device__ __forceinline__ float key_value(unsigned k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
// (key, id) as one number: larger comes first in the order
__device__ __forceinline__ u64 pair_of(unsigned key, unsigned id) { return ((u64)key << 32) | (0xffffffffu - id); }

struct Weigher {
  double m, c;          // largest logit, log2(e) / T
  unsigned mkey;
  bool top_inf;         // the largest logit is +inf: only its equals have weight
  const double* tab;
  // log2 of the weight (<= 0)
  __device__ __forceinline__ double exponent(unsigned key) const {
    if (key == mkey) return 0.0;
    if (top_inf) return -1e300;
    return ((double)key_value(key) - m) * c;
  }
  // the weight in units of 2^-45
  __device__ __forceinline__ u64 weight(double x) const {
    if (x < -SM_RANGE) return 0ull;
    const double t = x * 32.0, n = rint(t);
    const double r = (t - n) * 0.021660849392498290;      // ln 2 / 32; |r| <= ln 2 / 64
    double p = fma(r, 1.0 / 120.0, 1.0 / 24.0);           // exp(r), error r^6 / 720 <= 2.3e-15
    p = fma(r, p, 1.0 / 6.0);
    p = fma(r, p, 0.5);
    p = fma(r, p, 1.0);
    p = fma(r, p, 1.0);
    const int ni = (int)n;
    const double scale = __longlong_as_double((long long)(1023 + 45 + (ni >> 5)) << 52);
    return __double2ull_rn(tab[ni & 31] * p * scale);
  }
};

__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ u64 warp_max64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 t = __shfl_xor_sync(0xffffffffu, v, o);
    v = t > v ? t : v;
  }
  return v;
}

// floor(x * total) for x in [0, 1): exact for every x >= 2^-40
__device__ __forceinline__ u64 part_of(float x, u64 total) {
  if (!(x > 0.f)) return 0ull;
  return __umul64hi(__double2ull_rz((double)x * 18446744073709551616.0), total);
}

struct Cluster {
  cg::cluster_group cl;
  SampleShared* sh;
  int rank, S, phase, list;
  __device__ __forceinline__ SampleShared* peer(int r) { return S == 1 ? sh : cl.map_shared_rank(sh, r); }
  __device__ __forceinline__ void sync() {
    if (S == 1)
      __syncthreads();
    else
      cl.sync();
  }
  __device__ __forceinline__ void arrive() {
    if (S > 1) cl.barrier_arrive();
  }
  __device__ __forceinline__ void wait() {
    if (S > 1) cl.barrier_wait();
  }
  // every thread gets the values that thread 0 of every CTA gives: xch[return value][0..S)
  __device__ __forceinline__ int exchange(Sel v) {
    const int ph = phase;
    phase ^= 1;
    if (threadIdx.x < S) peer(threadIdx.x)->xch[ph][rank] = v;   // v is the same in every thread
    sync();
    return ph;
  }
};

enum { FIND_COUNT, FIND_MASS };

struct Row {
  const unsigned* keys;   // this CTA's part, shared memory
  int n, id0;             // its length and first id
};

// Gather the pairs that in_range takes (of all CTAs) into rank 0's list; returns how many there are.  Every CTA
// then holds a copy in cand[c.list] if they are at most SM_CAP.  Consecutive gathers use the two lists in turn, so
// a CTA may start the next one while another still ranks this one's; the other list's counter is cleared between
// this gather's two barriers, after its last reader and before its next writer.
template <class InRange>
__device__ unsigned gather(Cluster& c, const Row& row, InRange in_range) {
  SampleShared* lead = c.peer(0);
  const int q = c.list ^= 1;
  for (int i = threadIdx.x; i < row.n; i += SM_THREADS) {
    const unsigned key = row.keys[i];
    if (key == 0u) continue;
    const u64 pr = pair_of(key, row.id0 + i);
    if (in_range(key, pr)) {
      const unsigned at = atomicAdd(&lead->n_cand[q], 1u);
      if (at < SM_CAP) lead->cand[q][at] = pr;
    }
  }
  c.sync();
  const unsigned n = lead->n_cand[q];
  if (n <= SM_CAP && c.rank != 0)
    for (unsigned i = threadIdx.x; i < n; i += SM_THREADS) c.sh->cand[q][i] = lead->cand[q][i];
  if (c.rank == 0 && threadIdx.x == 0) c.sh->n_cand[q ^ 1] = 0u;
  c.sync();
  return n;
}

// The cut among n gathered pairs: the first whose mass (or count) up to and with it exceeds `target`.
// Every CTA computes the same.  0 if there is none.
__device__ u64 rank_candidates(Cluster& c, unsigned n, int mode, u64 target, const Weigher& w) {
  SampleShared* sh = c.sh;
  const u64* cand = sh->cand[c.list];
  u64 mine = 0ull, own = 0ull;
  __syncthreads();
  if (threadIdx.x == 0) sh->res_cut = 0ull;
  if (threadIdx.x < n) {
    mine = cand[threadIdx.x];
    own = mode == FIND_COUNT ? 1ull : w.weight(w.exponent((unsigned)(mine >> 32)));
    sh->cand_w[threadIdx.x] = own;
  }
  __syncthreads();
  if (threadIdx.x < n) {
    u64 before = 0ull;
    for (unsigned j = 0; j < n; ++j)
      if (cand[j] > mine) before += sh->cand_w[j];
    if (before <= target && before + own > target) sh->res_cut = mine;
  }
  __syncthreads();
  return sh->res_cut;
}

// Last element of the kept prefix among the pairs >= cut: the first one, in the order, whose count or mass up
// to and with it exceeds the target (count - 1, or top_p of the whole mass).  Returns `cut` if nothing does.
__device__ u64 find_cut(Cluster& c, const Row& row, const Weigher& w, int mode, u64 count_target, float top_p,
                        u64 cut, unsigned n_eligible) {
  SampleShared* sh = c.sh;
  if (n_eligible <= SM_CAP) {            // few enough to rank at once
    const unsigned n = gather(c, row, [&](unsigned, u64 pr) { return pr >= cut; });
    u64 target = count_target;
    if (mode == FIND_MASS) {
      u64 v = threadIdx.x < n ? w.weight(w.exponent((unsigned)(sh->cand[c.list][threadIdx.x] >> 32))) : 0ull;
      v = warp_sum64(v);
      __syncthreads();
      if ((threadIdx.x & 31) == 0) sh->wred[threadIdx.x >> 5] = v;
      __syncthreads();
      u64 total = 0ull;
      for (int i = 0; i < SM_WARPS; ++i) total += sh->wred[i];
      target = part_of(top_p, total);
    }
    const u64 r = rank_candidates(c, n, mode, target, w);
    return r ? r : cut;
  }
  // pass 0 bins by the exponent, later passes by the pair's bits in [lo, hi]
  u64 lo = 0ull, hi = ~0ull, target = count_target;
  int sh_bits = -1;
  for (int pass = 0; pass < 10; ++pass) {
    auto bin_of = [&](unsigned key, u64 pr, double x) -> int {
      if (sh_bits >= 0) return (int)((hi - pr) >> sh_bits);
      const float f = (float)(-x) * (float)((SM_BINS - 1) / SM_RANGE);
      return f < (float)(SM_BINS - 1) ? (int)f : SM_BINS - 1;
    };
    for (int i = threadIdx.x; i < 3 * SM_BINS; i += SM_THREADS) (&sh->hist[0][0])[i] = 0u;
    __syncthreads();
    unsigned tail = 0u;
    for (int i = threadIdx.x; i < row.n; i += SM_THREADS) {
      const unsigned key = row.keys[i];
      if (key == 0u) continue;
      const u64 pr = pair_of(key, row.id0 + i);
      if (pr < cut || pr < lo || pr > hi) continue;
      const double x = w.exponent(key);
      const int bin = bin_of(key, pr, x);
      if (mode == FIND_COUNT) {
        if (sh_bits < 0 && bin == SM_BINS - 1)
          ++tail;                        // the far tail is one bin: counted in registers
        else
          atomicAdd(&sh->hist[0][bin], 1u);
      } else {
        const u64 wt = w.weight(x);
        if (wt) {
          atomicAdd(&sh->hist[0][bin], (unsigned)(wt & 0xffffu));
          atomicAdd(&sh->hist[1][bin], (unsigned)((wt >> 16) & 0xffffu));
          atomicAdd(&sh->hist[2][bin], (unsigned)(wt >> 32));
        }
      }
    }
    if (mode == FIND_COUNT) {
      const unsigned t = __reduce_add_sync(0xffffffffu, tail);
      if ((threadIdx.x & 31) == 0 && t) atomicAdd(&sh->hist[0][SM_BINS - 1], t);
    }
    c.sync();
    // this CTA sums its share of the bins over the cluster: thread t has PB consecutive ones
    const int share = SM_BINS / c.S, b0 = c.rank * share;
    const int PB = (share + SM_THREADS - 1) / SM_THREADS;
    u64 val[SM_BINS / SM_THREADS], sum = 0ull;
#pragma unroll
    for (int q = 0; q < SM_BINS / SM_THREADS; ++q) {
      val[q] = 0ull;
      const int bl = threadIdx.x * PB + q;
      if (q < PB && bl < share)
        for (int r = 0; r < c.S; ++r) {
          const SampleShared* p = c.peer(r);
          val[q] += p->hist[0][b0 + bl];
          if (mode == FIND_MASS) val[q] += ((u64)p->hist[1][b0 + bl] << 16) + ((u64)p->hist[2][b0 + bl] << 32);
        }
      sum += val[q];
    }
    // exclusive prefix over the CTA's threads
    u64 inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 t = __shfl_up_sync(0xffffffffu, inc, o);
      if ((threadIdx.x & 31) >= o) inc += t;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 31) sh->wred[threadIdx.x >> 5] = inc;
    __syncthreads();
    u64 base = 0ull, mine = 0ull;
    for (int i = 0; i < SM_WARPS; ++i) {
      if (i < (int)(threadIdx.x >> 5)) base += sh->wred[i];
      mine += sh->wred[i];
    }
    if (threadIdx.x == 0) sh->res_bin = -1;
    const int ph = c.exchange(Sel{mine, 0ull});
    u64 total = 0ull;
    for (int r = 0; r < c.S; ++r) {
      if (r < c.rank) base += sh->xch[ph][r].a;
      total += sh->xch[ph][r].a;
    }
    if (mode == FIND_MASS && pass == 0) target = part_of(top_p, total);
    u64 at = base + inc - sum;
#pragma unroll
    for (int q = 0; q < SM_BINS / SM_THREADS; ++q) {
      if (at <= target && at + val[q] > target)
        for (int r = 0; r < c.S; ++r) {
          SampleShared* p = c.peer(r);
          p->res_bin = b0 + threadIdx.x * PB + q;
          p->res_base = at;
        }
      at += val[q];
    }
    c.sync();
    const int bin = sh->res_bin;
    if (bin < 0) return cut;             // everything is within the target
    target -= sh->res_base;
    u64 mn = ~0ull, mx = 0ull;
    const unsigned n = gather(c, row, [&](unsigned key, u64 pr) {
      if (pr < cut || pr < lo || pr > hi) return false;
      const bool in = bin_of(key, pr, sh_bits >= 0 ? 0.0 : w.exponent(key)) == bin;
      if (in) {
        mn = pr < mn ? pr : mn;
        mx = pr > mx ? pr : mx;
      }
      return in;
    });
    if (n <= SM_CAP) {
      const u64 r = rank_candidates(c, n, mode, target, w);
      return r ? r : cut;
    }
    // split the bin again: the range of the pairs that are in it
    mx = warp_max64(mx);
    mn = ~warp_max64(~mn);
    if ((threadIdx.x & 31) == 0) {
      sh->wred[threadIdx.x >> 5] = mx;
      sh->wred2[threadIdx.x >> 5] = mn;
    }
    __syncthreads();
    for (int i = 0; i < SM_WARPS; ++i) {
      mx = sh->wred[i] > mx ? sh->wred[i] : mx;
      mn = sh->wred2[i] < mn ? sh->wred2[i] : mn;
    }
    const int p2 = c.exchange(Sel{mx, mn});
    for (int r = 0; r < c.S; ++r) {
      mx = sh->xch[p2][r].a > mx ? sh->xch[p2][r].a : mx;
      mn = sh->xch[p2][r].b < mn ? sh->xch[p2][r].b : mn;
    }
    lo = mn;
    hi = mx;
    const int bits = 64 - __clzll((long long)(hi - lo));
    sh_bits = bits > 11 ? bits - 11 : 0;   // (hi - lo) >> sh_bits < 2048
  }
  return cut;                              // not reached: every pass leaves 1/2048 of a range of 2^64 pairs
}

template <bool F32>
__global__ void __launch_bounds__(SM_THREADS) sample_kernel(
    const void* __restrict__ logits, long long ld, int lim, int part, int stop_free, UtttSampling opt,
    const float* __restrict__ u, long long u_ld, const int* __restrict__ u_index, int u_len, int* __restrict__ ids,
    int* __restrict__ kept, float* __restrict__ prob) {
  extern __shared__ __align__(16) unsigned keys[];
  __shared__ SampleShared shared;
  SampleShared* sh = &shared;
  Cluster c{cg::this_cluster(), sh, (int)blockIdx.x, (int)gridDim.x, 0, 0};
  const int row_i = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  pdl_trigger();
  if (tid < 32) sh->tab[tid] = exp2((double)tid / 32.0);
  if (tid < 2) sh->n_cand[tid] = 0u;
  c.arrive();                            // peers write here only once every CTA of the cluster has started
  // ---- this CTA's part of the row, as keys
  Row row;
  row.keys = keys;
  row.id0 = c.rank * part;
  row.n = max(0, min(part, lim - row.id0));
  constexpr int E = F32 ? 4 : 8;         // logits per 16-byte load
  const char* src = reinterpret_cast<const char*>(logits) + ((size_t)row_i * ld + row.id0) * (F32 ? 4 : 2);
  u64 best = 0ull;
  unsigned count = 0u;
  auto put = [&](int i, unsigned bits) {
    const int id = row.id0 + i;
    const bool out = id == 0 || id == 1 || id == 3 || (stop_free && id < 6);
    const unsigned k = out ? 0u : order_key(bits);
    keys[i] = k;
    if (k) {
      ++count;
      const u64 pr = pair_of(k, id);
      best = pr > best ? pr : best;
    }
  };
  const int nv = (reinterpret_cast<uintptr_t>(src) & 15u) == 0 ? row.n / E : 0;
  for (int j = tid; j < nv; j += SM_THREADS) {
    const uint4 v = reinterpret_cast<const uint4*>(src)[j];
    const unsigned x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (F32) {
        put(j * E + e, x[e]);
      } else {
        put(j * E + 2 * e, x[e] << 16);
        put(j * E + 2 * e + 1, x[e] & 0xffff0000u);
      }
    }
  }
  for (int i = nv * E + tid; i < row.n; i += SM_THREADS)
    put(i, F32 ? reinterpret_cast<const unsigned*>(src)[i]
               : (unsigned)reinterpret_cast<const unsigned short*>(src)[i] << 16);
  best = warp_max64(best);
  count = __reduce_add_sync(0xffffffffu, count);
  if (lane == 0) {
    sh->wred[warp] = best;
    sh->wred2[warp] = count;
  }
  __syncthreads();
  u64 cnt = 0ull;
  for (int i = 0; i < SM_WARPS; ++i) {
    best = sh->wred[i] > best ? sh->wred[i] : best;
    cnt += sh->wred2[i];
  }
  c.wait();
  const int ph = c.exchange(Sel{best, cnt});
  cnt = 0ull;
  for (int r = 0; r < c.S; ++r) {
    best = sh->xch[ph][r].a > best ? sh->xch[ph][r].a : best;
    cnt += sh->xch[ph][r].b;
  }
  if (cnt == 0ull) {                     // nothing to choose from: an allowed id, as the greedy pick gives
    if (c.rank == 0 && tid == 0) {
      ids[row_i] = (stop_free ? 6 : 2) % lim;
      if (kept) kept[row_i] = 0;
      if (prob) prob[row_i] = 0.f;
    }
    c.sync();                            // no CTA leaves while a peer may still write to it
    return;
  }
  // ---- settings of the row
  float T = opt.temperature ? opt.temperature[row_i] : opt.temperature_all;
  const int top_k = opt.top_k ? opt.top_k[row_i] : opt.top_k_all;
  const float top_p = opt.top_p ? opt.top_p[row_i] : opt.top_p_all;
  const float min_p = opt.min_p ? opt.min_p[row_i] : opt.min_p_all;
  const bool greedy = !(T > SM_GREEDY_T) || top_k == 1;
  if (greedy) T = 1.f;
  Weigher w;
  w.mkey = (unsigned)(best >> 32);
  w.m = (double)key_value(w.mkey);
  w.top_inf = w.mkey == 0xff800000u;
  w.c = 1.4426950408889634074 / (double)T;
  w.tab = sh->tab;
  u64 cut = 0ull;
  if (greedy) {
    cut = best;
  } else {
    u64 eligible = cnt;
    if (top_k > 0 && (u64)top_k < cnt) {
      cut = find_cut(c, row, w, FIND_COUNT, (u64)(top_k - 1), 0.f, cut, (unsigned)eligible);
      eligible = top_k;
    }
    if (top_p < 1.f) cut = find_cut(c, row, w, FIND_MASS, 0ull, top_p, cut, (unsigned)eligible);
  }
  const double x_min = min_p > 0.f ? log2((double)fminf(min_p, 1.f)) : -INFINITY;
  // ---- mass of the kept elements per warp; warp k of the CTA has ids [k * seg, (k + 1) * seg) of its part
  const int seg = ((row.n + SM_WARPS - 1) / SM_WARPS + 31) & ~31;
  const int i0 = warp * seg, i1 = min(row.n, i0 + seg);
  auto weigh = [&](int i, bool& in) -> u64 {
    in = false;
    if (i >= i1) return 0ull;
    const unsigned key = keys[i];
    if (key == 0u || pair_of(key, row.id0 + i) < cut) return 0ull;
    const double x = w.exponent(key);
    if (!(x >= x_min)) return 0ull;
    in = true;
    return w.weight(x);
  };
  u64 mass = 0ull;
  count = 0u;
  for (int i = i0 + lane; i < i0 + seg; i += 32) {
    bool in;
    mass += weigh(i, in);
    count += in;
  }
  mass = warp_sum64(mass);
  count = __reduce_add_sync(0xffffffffu, count);
  __syncthreads();
  if (lane == 0) {
    sh->wred[warp] = mass;
    sh->wred2[warp] = count;
  }
  __syncthreads();
  u64 all = 0ull, below = 0ull;
  cnt = 0ull;
  for (int i = 0; i < SM_WARPS; ++i) {
    if (i < warp) below += sh->wred[i];
    all += sh->wred[i];
    cnt += sh->wred2[i];
  }
  const int p2 = c.exchange(Sel{all, cnt});
  u64 total = 0ull, n_kept = 0ull;
  for (int r = 0; r < c.S; ++r) {
    if (r < c.rank) below += sh->xch[p2][r].a;
    total += sh->xch[p2][r].a;
    n_kept += sh->xch[p2][r].b;
  }
  float uv = u[(size_t)row_i * u_ld + (u_index ? min(max(u_index[row_i], 0), u_len - 1) : 0)];
  uv = fminf(uv, 0.99999994f);           // the largest number below 1
  const u64 target = part_of(uv, total);
  if (below <= target && target < below + mass) {   // one warp of the cluster
    u64 at = below;
    for (int i = i0 + lane; i < i0 + seg; i += 32) {
      bool in;
      const u64 wt = weigh(i, in);
      u64 inc = wt;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 t = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += t;
      }
      const u64 tile = __shfl_sync(0xffffffffu, inc, 31);
      if (target < at + tile) {
        if (at + inc - wt <= target && target < at + inc) {
          ids[row_i] = row.id0 + i;
          if (kept) kept[row_i] = (int)n_kept;
          if (prob) prob[row_i] = (float)((double)wt / (double)total);
        }
        break;
      }
      at += tile;
    }
  }
  c.sync();                              // no CTA leaves while a peer may still read or write its shared memory
}

}  // namespace
}  // namespace uttt

using namespace uttt;

extern "C" int uttt_sample(int rows, int V, const void* logits, int logits_f32, long long ld, int active_limit,
                           int stop_free, const UtttSampling* opt, const float* u, long long u_ld,
                           const int* u_index, int u_len, int* ids, int* kept, float* prob, void* stream) {
  UTTT_REQUIRE(rows > 0 && V > 6 && logits && opt && u && ids && active_limit > 2, UTTT_ERR_INVALID);
  UTTT_REQUIRE(ld >= V && u_ld >= 0 && (!u_index || u_len > 0), UTTT_ERR_INVALID);
  UTTT_REQUIRE(V <= SM_MAX_V && rows <= 65535, UTTT_ERR_UNSUPPORTED);
  cudaStream_t st = (cudaStream_t)stream;
  ProfScope ps(UTTT_PROF_ARGMAX, st);
  const int lim = active_limit < V ? active_limit : V;
  // split a row over a cluster while the rows alone leave SMs idle (at least 1024 logits per CTA), or while
  // a CTA's part does not fit its shared memory
  int S = 1;
  while (S < SM_MAX_CTAS && ((lim + S - 1) / S > 32768 || ((long long)rows * S < num_sms() && lim / (2 * S) >= 1024)))
    S *= 2;
  const int part = ((lim + S - 1) / S + 7) & ~7;
  auto kernel = logits_f32 ? sample_kernel<true> : sample_kernel<false>;
  static DeviceOnce attr;
  UTTT_TRY(run_once_per_device(attr, [] {
    UTTT_TRY(cuda_status(cudaFuncSetAttribute(sample_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                              32768 * 4)));
    return cuda_status(cudaFuncSetAttribute(sample_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            32768 * 4));
  }));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(S, rows);
  cfg.blockDim = dim3(SM_THREADS);
  cfg.dynamicSmemBytes = (size_t)part * sizeof(unsigned);
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = S;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  at[1] = pdl_attribute();
  cfg.attrs = at;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, kernel, logits, ld, lim, part, stop_free, *opt, u, u_ld, u_index, u_len, ids, kept,
                         prob) != cudaSuccess)
    return launch_status();
  return launch_status();
}
