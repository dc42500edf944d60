// Sampling of one token per row from logits, with temperature, top-k, top-p and
// min-p, from one given uniform number per row (the rules of _sample_next_token,
// model/uttt_model.py:1181-1235, without its repetition penalty, plus top-k and min-p; the random number is an
// input, so a pick is repeatable whatever else is in the batch).
//
// Mathematics.  A row's candidates are its ids below active_limit that are not
// PAD / BOS / UNK and whose logit is neither NaN nor -inf.  With m the largest
// logit, w_i = exp((s_i - m) / T) = 2^-x_i, x_i = (m - s_i) log2(e) / T.  Candidates
// are ordered by (s descending, id ascending); top-k keeps the first k, top-p
// those whose mass before them is at most top_p times the mass top-k left, min-p
// those with w_i >= min_p.  All three keep a prefix of that order, so the kept set
// is one cut element.  The pick is the lowest id i with (sum of kept w_j, j <= i)
// > u * (sum of all kept w_j).
//
// Whole-number weights.  x_i is computed in 64 bits and split into the nearest k / 128
// and the rest; 2^-x_i comes from the integer part of k / 128 (the exponent), the
// other 7 bits of k (a table of 2^(-j/128)) and the rest (a cubic Taylor polynomial:
// the table-driven method of Tang, ACM TOMS 15, 1989), good to 2^-38 of itself and
// rounded to a whole number of 2^-45.  Weights below 2^-24 take x and 2^-x from FP32
// instead: off by 2^-19 of themselves, they are still good to 2^-43 of the largest.
// So every sum of weights is an exact integer (64-bit, or in a double while it is
// below 2^53) that does not depend on the order of the additions: histograms with
// atomics, splits over CTAs and any grid give the same cut and the same pick.
// 64-bit floating point, because its pipe is idle: with the same steps in 32-bit
// integers the half-rate integer pipe was 60 % busy and bound the kernel.
//
// Layout.  One cluster of S CTAs per row; each warp owns a contiguous piece of the
// row and streams it in 16-byte loads, once per step (the row comes from HBM once;
// a small piece then stays in shared memory, others come from L2 again):
// (1) largest logit; (2) where top-k or top-p ask for it, a histogram over 2048 bins
// of x, merged over the cluster in distributed shared memory; (3) where the
// candidates down to the cut's bin are few, all of them in one list, from which the
// row is finished; else those of the bin, ranked against each other (of too many
// equal logits the last kept one is counted off in id order, and a bin with too many
// nearly equal ones is split again by the bits of its (key, id) pairs); (4) kept mass
// per warp; the CTA that holds the pick weighs that warp's piece again.  Weights below
// 2^-24 (a billionth of a percent of the mass each) get no bin: what top-p asks for
// nearly always ends before them, and if it does not, they are one bin that is split
// by the same steps.
//
// What bounds it.  Large batches: instructions.  256 rows of 131072 BF16 logits at
// top-p 0.95 take 196 us, 140 warp instructions per 32 logits over the four walks at
// 0.73 a cycle and scheduler (FP64 14 %, ALU 44 %, DRAM 4 % busy): 8 % of the time for
// the largest logit, 42 % for the histogram, 13 % for the gather, 31 % for the kept
// mass.  Without cuts they take 100 us.  Small ones: latency, 7 cluster barriers and
// more walks the more is kept.  In a row of calls a row of 32000 FP32 logits takes 17 us
// at T 0.7, top-p 0.9 (5 ids kept, finished in the list) and 21 at T 1, top-p 0.95
// (6200 kept; 32 alone); 64 rows 17 us at top-k 50 and 30 at top-p 0.95; 333 rows of
// 8003 24 and 43 (38 for rows of 8000, which all start on 16 bytes).
#include <cooperative_groups.h>

#include "common.cuh"
#include "host_util.cuh"

namespace cg = cooperative_groups;

namespace uttt {
namespace {

constexpr int SM_THREADS = 512;
constexpr int SM_WARPS = SM_THREADS / 32;
constexpr int SM_BINS = 2048;
constexpr int SM_CAP = SM_THREADS;        // candidates ranked against each other directly, one per thread
constexpr int SM_RING = 4;               // 16-byte vectors on their way per lane
constexpr int SM_TAIL = SM_BINS;          // the bin of everything beyond SM_RANGE
constexpr int SM_MAX_CTAS = 8;
constexpr int SM_MAX_V = 262144;
constexpr int SM_MAX_PART = 131071;      // candidates per CTA: sums of as many limbs of up to 2^15 stay below 2^32
constexpr int SM_MAX_VECS = 16384;       // 8-logit vectors per CTA: 1024 a warp, so a lane adds at most 256 weights
constexpr float SM_RANGE = 24.f;         // x up to here has bins (64 to the unit) and exact weights
constexpr int SM_STEPS = 128;            // table entries per octave
constexpr float SM_GREEDY_T = 1e-5f;     // _sample_next_token's greedy border

typedef unsigned long long u64;

struct Sel {     // value exchanged between the CTAs of a cluster
  u64 a, b;
};

struct SampleShared {
  uint4 ring[SM_WARPS][SM_RING * 32];    // vectors on their way
  double tab[SM_STEPS * 16];             // the table 16 times: the lanes of a half-warp meet no bank conflicts
  Sel xch[2][SM_MAX_CTAS];               // one slot per CTA, two phases
  u64 wred[SM_WARPS], wred2[SM_WARPS];
  u64 found[2][SM_CAP];                  // this CTA's gathered candidates; gathers alternate between the two lists
  u64 cand[SM_CAP], cand_w[SM_CAP];      // the whole cluster's, and their weights
  unsigned n_found[2];
  u64 res_base, res_held, res_cut;
  int res_bin;
  u64 more[SM_MAX_CTAS * SM_WARPS];      // what every warp of the cluster has beyond the bins
  alignas(16) unsigned hist[3][SM_BINS];  // count, or 15-bit limbs of the mass
  alignas(16) u64 merged[SM_BINS];       // the cluster's histogram
};

// 2^45 * 2^(-j / 128)
__device__ const double kPow2[SM_STEPS] = {
    0x1.0000000000000p+45, 0x1.fd3c22b8f71f1p+44, 0x1.fa7c1819e90d8p+44, 0x1.f7bfdad9cbe14p+44,
    0x1.f50765b6e4540p+44, 0x1.f252b376bba97p+44, 0x1.efa1bee615a27p+44, 0x1.ecf482d8e67f1p+44,
    0x1.ea4afa2a490dap+44, 0x1.e7a51fbc74c83p+44, 0x1.e502ee78b3ff6p+44, 0x1.e264614f5a129p+44,
    0x1.dfc97337b9b5fp+44, 0x1.dd321f301b460p+44, 0x1.da9e603db3285p+44, 0x1.d80e316c98398p+44,
    0x1.d5818dcfba487p+44, 0x1.d2f87080d89f2p+44, 0x1.d072d4a07897cp+44, 0x1.cdf0b555dc3fap+44,
    0x1.cb720dcef9069p+44, 0x1.c8f6d9406e7b5p+44, 0x1.c67f12e57d14bp+44, 0x1.c40ab5fffd07ap+44,
    0x1.c199bdd85529cp+44, 0x1.bf2c25bd71e09p+44, 0x1.bcc1e904bc1d2p+44, 0x1.ba5b030a1064ap+44,
    0x1.b7f76f2fb5e47p+44, 0x1.b59728de5593ap+44, 0x1.b33a2b84f15fbp+44, 0x1.b0e07298db666p+44,
    0x1.ae89f995ad3adp+44, 0x1.ac36bbfd3f37ap+44, 0x1.a9e6b5579fdbfp+44, 0x1.a799e1330b358p+44,
    0x1.a5503b23e255dp+44, 0x1.a309bec4a2d33p+44, 0x1.a0c667b5de565p+44, 0x1.9e86319e32323p+44,
    0x1.9c49182a3f090p+44, 0x1.9a0f170ca07bap+44, 0x1.97d829fde4e50p+44, 0x1.95a44cbc8520fp+44,
    0x1.93737b0cdc5e5p+44, 0x1.9145b0b91ffc6p+44, 0x1.8f1ae99157736p+44, 0x1.8cf3216b5448cp+44,
    0x1.8ace5422aa0dbp+44, 0x1.88ac7d98a6699p+44, 0x1.868d99b4492edp+44, 0x1.8471a4623c7adp+44,
    0x1.82589994cce13p+44, 0x1.80427543e1a12p+44, 0x1.7e2f336cf4e62p+44, 0x1.7c1ed0130c132p+44,
    0x1.7a11473eb0187p+44, 0x1.780694fde5d3fp+44, 0x1.75feb564267c9p+44, 0x1.73f9a48a58174p+44,
    0x1.71f75e8ec5f74p+44, 0x1.6ff7df9519484p+44, 0x1.6dfb23c651a2fp+44, 0x1.6c012750bdabfp+44,
    0x1.6a09e667f3bcdp+44, 0x1.68155d44ca973p+44, 0x1.6623882552225p+44, 0x1.6434634ccc320p+44,
    0x1.6247eb03a5585p+44, 0x1.605e1b976dc09p+44, 0x1.5e76f15ad2148p+44, 0x1.5c9268a5946b7p+44,
    0x1.5ab07dd485429p+44, 0x1.58d12d497c7fdp+44, 0x1.56f4736b527dap+44, 0x1.551a4ca5d920fp+44,
    0x1.5342b569d4f82p+44, 0x1.516daa2cf6642p+44, 0x1.4f9b2769d2ca7p+44, 0x1.4dcb299fddd0dp+44,
    0x1.4bfdad5362a27p+44, 0x1.4a32af0d7d3dep+44, 0x1.486a2b5c13cd0p+44, 0x1.46a41ed1d0057p+44,
    0x1.44e086061892dp+44, 0x1.431f5d950a897p+44, 0x1.4160a21f72e2ap+44, 0x1.3fa4504ac801cp+44,
    0x1.3dea64c123422p+44, 0x1.3c32dc313a8e5p+44, 0x1.3a7db34e59ff7p+44, 0x1.38cae6d05d866p+44,
    0x1.371a7373aa9cbp+44, 0x1.356c55f929ff1p+44, 0x1.33c08b26416ffp+44, 0x1.32170fc4cd831p+44,
    0x1.306fe0a31b715p+44, 0x1.2ecafa93e2f56p+44, 0x1.2d285a6e4030bp+44, 0x1.2b87fd0dad990p+44,
    0x1.29e9df51fdee1p+44, 0x1.284dfe1f56381p+44, 0x1.26b4565e27cddp+44, 0x1.251ce4fb2a63fp+44,
    0x1.2387a6e756238p+44, 0x1.21f49917ddc96p+44, 0x1.2063b88628cd6p+44, 0x1.1ed5022fcd91dp+44,
    0x1.1d4873168b9aap+44, 0x1.1bbe084045cd4p+44, 0x1.1a35beb6fcb75p+44, 0x1.18af9388c8deap+44,
    0x1.172b83c7d517bp+44, 0x1.15a98c8a58e51p+44, 0x1.1429aaea92de0p+44, 0x1.12abdc06c31ccp+44,
    0x1.11301d0125b51p+44, 0x1.0fb66affed31bp+44, 0x1.0e3ec32d3d1a2p+44, 0x1.0cc922b7247f7p+44,
    0x1.0b5586cf9890fp+44, 0x1.09e3ecac6f383p+44, 0x1.0874518759bc8p+44, 0x1.0706b29ddf6dep+44,
    0x1.059b0d3158574p+44, 0x1.04315e86e7f85p+44, 0x1.02c9a3e778061p+44, 0x1.0163da9fb3335p+44,
};

// order-preserving key of a logit: larger logit, larger key.  Both zeros are one value.
__device__ __forceinline__ unsigned order_key(unsigned bits) {
  const unsigned k = bits ^ ((unsigned)((int)bits >> 31) | 0x80000000u);
  return k == 0x7fffffffu ? 0x80000000u : k;
}
// whether a key is a candidate's: neither NaN (beyond either end) nor -inf
__device__ __forceinline__ bool is_candidate(unsigned k) { return k - 0x00800000u <= 0xff000000u; }
constexpr unsigned kInfKey = 0xff800000u;   // of +inf, the largest candidate
__device__ __forceinline__ float key_value(unsigned k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
// (key, id) as one number: larger comes first in the order
__device__ __forceinline__ u64 pair_of(unsigned key, unsigned id) { return ((u64)key << 32) | (0xffffffffu - id); }

// Rows with +inf among their logits: only the infinities have weight (the others' is exp(-inf)).  +inf is taken as the
// largest finite number and that one, in such a row, as the number below it, whose distance of 2^104 leaves no weight.
constexpr float kMaxFinite = 3.402823466e+38f;
__device__ __forceinline__ unsigned finite_top(unsigned bits) {
  return bits == 0x7f800000u || bits == 0x7f7fffffu ? bits - 1u : bits;
}

// an integer in 0 .. 2^52 - 1 that was added to 2^52
__device__ __forceinline__ u64 mantissa(double v) {
  return ((u64)((unsigned)__double2hiint(v) & 0xfffffu) << 32) | (unsigned)__double2loint(v);
}

struct Weigher {
  double m, c;          // largest logit, 128 log2(e) / T
  float scale, ms, cs;  // a power of 2, m times it, and log2(e) / T divided by it
  const double* tab;    // this lane's copy
  // x in FP32; NaN or infinite for NaN and -inf.  Scaled, so that m - s does not overflow: by 1/2, and by 2^-100 at
  // temperatures above 10^30, which would flush log2(e) / T to zero
  __device__ __forceinline__ float rough(unsigned bits) const { return fmaf(__uint_as_float(bits), -scale, ms) * cs; }
  // logits for quick tests: none whose x is at most y is smaller, or at least y larger
  __device__ __forceinline__ float no_less(float y) const {
    return __double2float_rd(m - ((double)y * 1.000001 + 1e-5) / ((double)cs * (double)scale));
  }
  __device__ __forceinline__ float no_more(float y) const {
    return __double2float_ru(m - ((double)y * 0.999999 - 1e-5) / ((double)cs * (double)scale));
  }
  // m - s >= 0, exact but for one rounding to 53 bits
  __device__ __forceinline__ double below(unsigned bits) const { return m - (double)__uint_as_float(bits); }
  // k, the whole number next to 128 x, and the rest r
  __device__ __forceinline__ int split(double d, double& r) const {
    constexpr double magic = 6755399441055744.0;         // 1.5 * 2^52: the last place is 1
    const double t = fma(d, c, magic);
    r = fma(d, c, magic - t);
    return __double2loint(t);
  }
  __device__ __forceinline__ int bin(int k) const { return k >> 1; }   // 64 to the unit
  // 2^52 + 2^-x in units of 2^-45, rounded
  __device__ __forceinline__ double weight52(int k, double r) const {
    const double t = tab[(k & (SM_STEPS - 1)) * 16];
    // 2^(-r / 128), |r| <= 1/2: the next term of the series is below 2^-38
    const double p = fma(r, fma(r, fma(r, -2.646642144433097e-08, 1.4662262387640425e-05), -0.0054152123481245725), 1.0);
    const double scaled = __hiloint2double(__double2hiint(t) - (k >> 7) * 0x100000, __double2loint(t));
    return fma(scaled, p, 4503599627370496.0);
  }
  // 2^-x in units of 2^-45 for rough x > SM_RANGE (0 for NaN and infinities): below 2^21, so that adding 2^23 rounds it
  // to a whole number in the mantissa
  __device__ __forceinline__ unsigned tail_weight(float y) const {
    return y < 64.f ? __float_as_uint(exp2f(45.f - y) + 8388608.f) & 0x7fffffu : 0u;
  }
  __device__ __forceinline__ u64 weight_of(unsigned bits) const {
    const float y = rough(bits);
    if (!(y <= SM_RANGE)) return (u64)tail_weight(y);
    double r;
    const int k = split(below(bits), r);
    return mantissa(weight52(k, r));
  }
  // the same by key
  __device__ __forceinline__ u64 weight_of_key(unsigned key) const { return weight_of(__float_as_uint(key_value(key))); }
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

// the largest number, subnormal ones too (the compiler's own flag would flush them); a NaN loses
__device__ __forceinline__ float max_exact(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Sums over the CTA's warps of two numbers that every lane of a warp has, and the first one's over the warps before
// this one.  Each warp adds its 16 numbers by shuffles: read one by one they are 16 warps' worth of issue slots.
struct Sums {
  u64 a, b, a_below;
};
__device__ __forceinline__ Sums block_sums(SampleShared* sh, u64 a, u64 b) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, w = lane & (SM_WARPS - 1);
  __syncthreads();
  if (lane == 0) {
    sh->wred[warp] = a;
    sh->wred2[warp] = b;
  }
  __syncthreads();
  Sums s{sh->wred[w], sh->wred2[w], 0ull};
  if (w < warp) s.a_below = s.a;
#pragma unroll
  for (int o = SM_WARPS / 2; o > 0; o >>= 1) {
    s.a += __shfl_xor_sync(0xffffffffu, s.a, o);
    s.b += __shfl_xor_sync(0xffffffffu, s.b, o);
    s.a_below += __shfl_xor_sync(0xffffffffu, s.a_below, o);
  }
  return s;
}

// floor(x * total) for x in [0, 1): exact for every x >= 2^-40
__device__ __forceinline__ u64 part_of(float x, u64 total) {
  if (!(x > 0.f)) return 0ull;
  return __umul64hi(__double2ull_rz((double)x * 18446744073709551616.0), total);
}

struct Cluster {
  cg::cluster_group cl;
  SampleShared* sh;
  int rank, S, phase, list;              // list: of the last gather
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
    if ((int)threadIdx.x < S) peer(threadIdx.x)->xch[ph][rank] = v;   // v is the same in every thread
    sync();
    return ph;
  }
  // sums of what the CTAs gave, and the first one's over the CTAs before this one
  __device__ __forceinline__ Sums sums(int ph) const {
    const int r = threadIdx.x & (SM_MAX_CTAS - 1);
    Sums s{0ull, 0ull, 0ull};
    if (r < S) {
      s.a = sh->xch[ph][r].a;
      s.b = sh->xch[ph][r].b;
      if (r < rank) s.a_below = s.a;
    }
#pragma unroll
    for (int o = SM_MAX_CTAS / 2; o > 0; o >>= 1) {
      s.a += __shfl_xor_sync(0xffffffffu, s.a, o);
      s.b += __shfl_xor_sync(0xffffffffu, s.b, o);
      s.a_below += __shfl_xor_sync(0xffffffffu, s.a_below, o);
    }
    return s;
  }
};

enum { FIND_COUNT, FIND_MASS };

// 8 logits from id i on, one by one (rows that do not start on 16 bytes, and the end of a row)
struct Eight {
  unsigned x[8];
};
template <bool F32>
__device__ __noinline__ Eight load_scalar(const char* src, int i, int V) {
  Eight r;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int k = min(i + e, V - 1);     // what lies behind the row is masked by the caller
    r.x[e] = F32 ? reinterpret_cast<const unsigned*>(src)[k]
                 : (unsigned)reinterpret_cast<const unsigned short*>(src)[k] << 16;
  }
  return r;
}

// A row's piece of one warp: 8-logit vectors v0 .. v1 - 1, the lanes side by side.
template <bool F32>
struct Row {
  const char* src;        // the row
  bool vec;               // whether it starts on 16 bytes
  bool has_inf;           // whether its largest logit is +inf
  bool kept;              // whether the whole piece is in the ring, from an earlier walk
  int V, lim, stop_free;
  int v0, v1;
  uint4* ring;            // the warp's places in shared memory

  // f(bits[8], first id) for every vector of the piece, in step over the warp, until it returns false; ids that are
  // never picked come as -inf.  Vectors arrive by cp.async, each lane's own ones in its own places, a few ahead; a
  // piece of no more vectors than places stays there for the walks after the first.
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    const int lane = threadIdx.x & 31;
    constexpr int ahead = F32 ? SM_RING / 2 : SM_RING;
    constexpr int W = F32 ? 2 : 1;       // 16-byte pieces of a vector
    uint4* const mine = ring + lane;
    const uint4* next = reinterpret_cast<const uint4*>(src) + (size_t)(v0 + lane) * W;
    const int full = vec ? min(v1, V / 8) : 0;   // vectors that can be fetched whole
    int vf = v0 + lane;                  // the next one to fetch, into place sf
    unsigned sf = 0;
    auto fetch = [&]() {
      if (vf < full) {
        cp_async_16(mine + sf * (W * 32), next, true);
        if (F32) cp_async_16(mine + sf * (W * 32) + 32, next + 1, true);
      }
      cp_async_commit();
      next += 32 * W;
      vf += 32;
      sf = (sf + 1) & (ahead - 1);
    };
    if (!kept) {
#pragma unroll 1
      for (int k = 0; k < ahead - 1; ++k) fetch();
    }
    unsigned sr = 0;
#pragma unroll 1
    for (int t = v0; t < v1; t += 32) {
      const int v = t + lane;
      if (!kept) {
        fetch();
        cp_async_wait<ahead - 1>();
      }
      unsigned x[8];
      const uint4* at = mine + sr * (W * 32);
      sr = (sr + 1) & (ahead - 1);
      if (v < full) {
        const uint4 a = at[0];
        if (F32) {
          const uint4 b = at[32];
          x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        } else {
          x[0] = a.x << 16, x[1] = a.x & 0xffff0000u, x[2] = a.y << 16, x[3] = a.y & 0xffff0000u;
          x[4] = a.z << 16, x[5] = a.z & 0xffff0000u, x[6] = a.w << 16, x[7] = a.w & 0xffff0000u;
        }
      } else {
        const Eight r = load_scalar<F32>(src, min(v, v1 - 1) * 8, V);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = r.x[e];
      }
      if (has_inf) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = finite_top(x[e]);
      }
      if (v == 0 || v >= v1 || v * 8 + 8 > lim) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int id = v * 8 + e;
          if (v >= v1 || id >= lim || id == 0 || id == 1 || id == 3 || (stop_free && id < 6)) x[e] = 0xff800000u;
        }
      }
      if (!f(x, v * 8)) break;
    }
    cp_async_wait<0>();                  // the places are free for the next walk
  }
};

__device__ __forceinline__ unsigned nth_of(const unsigned (&x)[8], int e) {
  unsigned r = x[0];
#pragma unroll
  for (int k = 1; k < 8; ++k) r = e == k ? x[k] : r;
  return r;
}

// Gather the pairs that in_range(bits, id) takes, of all CTAs; returns how many there are.  near(bits) is a quick test
// that lets all of them pass and few others.  Every CTA gathers its own in a list and, if they are at most SM_CAP in
// all, copies the cluster's lists into cand.  Consecutive gathers use the two lists in turn, so a CTA may start the next
// one while another still copies; the other list's counter is cleared behind this gather's barrier, after its last
// reader and before its next writer.
template <bool F32, class Near, class InRange>
__device__ unsigned gather(Cluster& c, const Row<F32>& row, Near near, InRange in_range) {
  SampleShared* sh = c.sh;
  const int q = c.list ^= 1;
  row.each([&](const unsigned (&x)[8], int id) {
    unsigned mask = 0u;
#pragma unroll
    for (int e = 0; e < 8; ++e) mask |= near(x[e]) ? 1u << e : 0u;
    for (; mask; mask &= mask - 1) {
      const int e = __ffs((int)mask) - 1;
      const unsigned xe = nth_of(x, e);
      if (in_range(xe, id + e)) {
        const unsigned at = atomicAdd(&sh->n_found[q], 1u);
        if (at < SM_CAP) sh->found[q][at] = pair_of(order_key(xe), id + e);
      }
    }
    return true;
  });
  c.sync();
  unsigned n = 0u, from = 0u, mine = 0u;   // cand[threadIdx.x] is number `mine` of CTA `from`
#pragma unroll
  for (int r = 0; r < SM_MAX_CTAS; ++r)
    if (r < c.S) {
      const unsigned k = c.peer(r)->n_found[q];
      if (threadIdx.x >= n) {
        from = r;
        mine = threadIdx.x - n;
      }
      n += k;
    }
  if (threadIdx.x < n && n <= SM_CAP) sh->cand[threadIdx.x] = c.peer(from)->found[q][mine];
  if (threadIdx.x == 0) sh->n_found[q ^ 1] = 0u;
  __syncthreads();
  return n;
}

// The cut among n gathered pairs: the first whose mass (or count) up to and with it exceeds `target`.
// Every CTA computes the same.  0 if there is none.
__device__ u64 rank_candidates(Cluster& c, unsigned n, int mode, u64 target, const Weigher& w) {
  SampleShared* sh = c.sh;
  const u64* cand = sh->cand;
  u64 mine = 0ull, own = 0ull;
  __syncthreads();
  if (threadIdx.x == 0) sh->res_cut = 0ull;
  if (threadIdx.x < n) {
    mine = cand[threadIdx.x];
    own = mode == FIND_COUNT ? 1ull : w.weight_of_key((unsigned)(mine >> 32));
    sh->cand_w[threadIdx.x] = own;
  }
  __syncthreads();
  if (threadIdx.x < n) {
    u64 before = 0ull;
#pragma unroll 8
    for (unsigned j = 0; j < n; ++j) before += cand[j] > mine ? sh->cand_w[j] : 0ull;
    if (before <= target && before + own > target) sh->res_cut = mine;
  }
  __syncthreads();
  return sh->res_cut;
}

// This CTA's share of the bins, added up over a cluster of S and sent to all of it.  All loads are in flight together
// (under a test of S each waited for the one before it: 6500 cycles for 8 CTAs).
template <int S>
__device__ __forceinline__ void merge_bins(Cluster& c, int mode) {
  SampleShared* p[S];
#pragma unroll
  for (int r = 0; r < S; ++r) p[r] = c.cl.map_shared_rank(c.sh, r);
  for (int i = threadIdx.x; i < SM_BINS / S; i += SM_THREADS) {
    const int bin = c.rank * (SM_BINS / S) + i;
    unsigned h0[S], h1[S], h2[S];
#pragma unroll
    for (int r = 0; r < S; ++r) h0[r] = p[r]->hist[0][bin];
    u64 v = 0ull;
    if (mode == FIND_MASS) {
#pragma unroll
      for (int r = 0; r < S; ++r) {
        h1[r] = p[r]->hist[1][bin];
        h2[r] = p[r]->hist[2][bin];
      }
#pragma unroll
      for (int r = 0; r < S; ++r) v += ((u64)h1[r] << 15) + ((u64)h2[r] << 30);
    }
#pragma unroll
    for (int r = 0; r < S; ++r) v += h0[r];
#pragma unroll
    for (int r = 0; r < S; ++r) p[r]->merged[bin] = v;
  }
}

// The cluster's histogram's bin that holds `target`, what lies before it and what is in it, the same in every CTA;
// `total`: of all bins.  With top_p > 0 the target is that part of total + more (mass), and written back.  The bin is -1
// if the target lies behind all bins.  Every CTA adds up its share of the bins over the cluster and sends the sums to
// all, who then look for the bin each: two cluster barriers, and remote loads that are in flight together.
__device__ int locate(Cluster& c, int mode, float top_p, u64 more, u64& target, u64& base_out, u64& held,
                      u64& total) {
  SampleShared* sh = c.sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int Q = SM_BINS / SM_THREADS;
  u64 val[Q];
  more = warp_sum64(more);
  c.sync();
  if (c.S == 1) {
    const uint4 h0 = reinterpret_cast<const uint4*>(sh->hist[0])[tid];
    val[0] = h0.x, val[1] = h0.y, val[2] = h0.z, val[3] = h0.w;
    if (mode == FIND_MASS) {
      const uint4 h1 = reinterpret_cast<const uint4*>(sh->hist[1])[tid], h2 = reinterpret_cast<const uint4*>(sh->hist[2])[tid];
      val[0] += ((u64)h1.x << 15) + ((u64)h2.x << 30), val[1] += ((u64)h1.y << 15) + ((u64)h2.y << 30);
      val[2] += ((u64)h1.z << 15) + ((u64)h2.z << 30), val[3] += ((u64)h1.w << 15) + ((u64)h2.w << 30);
    }
  } else {
    if (c.S == 2) merge_bins<2>(c, mode);
    if (c.S == 4) merge_bins<4>(c, mode);
    if (c.S == 8) merge_bins<8>(c, mode);
    if (lane < c.S) c.peer(lane)->more[c.rank * SM_WARPS + warp] = more;
    c.sync();
    const ulonglong2* m = reinterpret_cast<const ulonglong2*>(sh->merged) + tid * (Q / 2);
#pragma unroll
    for (int q = 0; q < Q; q += 2) {
      val[q] = m[q / 2].x;
      val[q + 1] = m[q / 2].y;
    }
    more = 0ull;
    for (int i = lane; i < c.S * SM_WARPS; i += 32) more += sh->more[i];
    more = warp_sum64(more);
  }
  u64 sum = 0ull;
#pragma unroll
  for (int q = 0; q < Q; ++q) sum += val[q];
  u64 inc = sum;                         // prefix over the threads
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 t = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += t;
  }
  if (tid == 0) sh->res_bin = -1;
  const Sums s = block_sums(sh, __shfl_sync(0xffffffffu, inc, 31), more);
  total = s.a;
  if (c.S == 1) more = s.b;
  if (top_p > 0.f) target = part_of(top_p, total + more);
  u64 at = s.a_below + inc - sum;
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    if (at <= target && at + val[q] > target) {
      sh->res_bin = tid * Q + q;
      sh->res_base = at;
      sh->res_held = val[q];
    }
    at += val[q];
  }
  __syncthreads();
  base_out = sh->res_base;
  held = sh->res_held;
  return sh->res_bin;
}

__device__ __forceinline__ void add_mass(SampleShared* sh, int bin, u64 wt) {
  const unsigned l0 = (unsigned)wt & 0x7fffu, l1 = (unsigned)(wt >> 15) & 0x7fffu, l2 = (unsigned)(wt >> 30);   // <= 2^15
  atomicAdd(&sh->hist[0][bin], l0);
  atomicAdd(&sh->hist[1][bin], l1);
  if (l2) atomicAdd(&sh->hist[2][bin], l2);
}

__device__ __forceinline__ void clear_hist(SampleShared* sh) {
  uint4* h = reinterpret_cast<uint4*>(&sh->hist[0][0]);
  for (int i = threadIdx.x; i < 3 * SM_BINS / 4; i += SM_THREADS) h[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
}

// The pair of the n-th (from 0, by id) candidate with this key; there are more than n of them.  One exchange (on a
// copy of c).
template <bool F32>
__device__ __noinline__ u64 nth_equal(Cluster c, const Row<F32> row, unsigned key, u64 n) {
  SampleShared* sh = c.sh;
  const int lane = threadIdx.x & 31;
  unsigned count = 0u;
  row.each([&](const unsigned (&x)[8], int) {
#pragma unroll
    for (int e = 0; e < 8; ++e) count += order_key(x[e]) == key;
    return true;
  });
  count = __reduce_add_sync(0xffffffffu, count);
  const Sums in = block_sums(sh, count, 0ull);
  const u64 below = in.a_below + c.sums(c.exchange(Sel{in.a, 0ull})).a_below;
  if (below <= n && n < below + count) {   // one warp of the cluster
    u64 at = below;
    row.each([&](const unsigned (&x)[8], int id) {
      unsigned mine = 0u;
#pragma unroll
      for (int e = 0; e < 8; ++e) mine += order_key(x[e]) == key;
      unsigned inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned t = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += t;
      }
      const unsigned tile = __shfl_sync(0xffffffffu, inc, 31);
      if (n >= at + tile) {
        at += tile;
        return true;
      }
      u64 run = at + inc - mine;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (order_key(x[e]) == key && run++ == n)
          for (int r = 0; r < c.S; ++r) c.peer(r)->res_cut = pair_of(key, id + e);
      return false;
    });
  }
  c.sync();
  return sh->res_cut;
}

// Last element of the kept prefix among the pairs >= cut: the first one, in the order, whose count or mass up
// to and with it exceeds the target (count - 1, or top_p of the whole mass).  Returns `cut` if nothing does.
// Where the candidates down to the cut are few and `cut` is 0, they are gathered as a whole instead: `listed` says how
// many are in the list (0: there is none, and the cut is returned), `target` what they must not exceed.
template <int MODE, bool F32>
__device__ u64 find_cut(Cluster& c, const Row<F32>& row, const Weigher& w, u64& target, float top_p, u64 cut,
                        unsigned n_eligible, unsigned& listed) {
  SampleShared* sh = c.sh;
  if (n_eligible <= SM_CAP) {            // few enough to rank at once
    const unsigned cut_bits = __float_as_uint(key_value((unsigned)(cut >> 32)));
    const float least = cut ? __uint_as_float(cut_bits) : -INFINITY;
    const unsigned n = gather(
        c, row, [&](unsigned bits) { return __uint_as_float(bits) >= least; },
        [&](unsigned bits, int id) {
          const unsigned key = order_key(bits);
          return is_candidate(key) && pair_of(key, id) >= cut;
        });
    if (MODE == FIND_MASS) {
      const u64 v = threadIdx.x < n ? w.weight_of_key((unsigned)(sh->cand[threadIdx.x] >> 32)) : 0ull;
      target = part_of(top_p, block_sums(sh, warp_sum64(v), 0ull).a);
    }
    if (cut == 0ull) {
      listed = n;
      return 0ull;
    }
    const u64 r = rank_candidates(c, n, MODE, target, w);
    return r ? r : cut;
  }
  clear_hist(sh);
  u64 more = 0ull, base, total;
  const unsigned cut_key = (unsigned)(cut >> 32);
  row.each([&](const unsigned (&x)[8], int id) {
    unsigned tail = 0u;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float y = w.rough(x[e]);
      if (cut_key) {                     // a cut from top-k
        const unsigned key = order_key(x[e]);
        if (key < cut_key || pair_of(key, id + e) < cut) continue;
      }
      if (y <= SM_RANGE) {
        double r;
        const int k = w.split(w.below(x[e]), r);
        if (MODE == FIND_COUNT)
          atomicAdd(&sh->hist[0][w.bin(k)], 1u);
        else
          add_mass(sh, w.bin(k), mantissa(w.weight52(k, r)));
      } else if (MODE == FIND_MASS) {
        tail += w.tail_weight(y);
      }
    }
    more += tail;
    return true;
  });
  u64 held;
  int bin = locate(c, MODE, MODE == FIND_MASS ? top_p : 0.f, more, target, base, held, total);
  if (bin < 0) {
    bin = SM_TAIL;
    base = total;
  }
  if (bin != SM_TAIL && cut == 0ull) {
    // an upper bound of the candidates down to this bin's end: each weighs at least 2^-x there
    const u64 least = MODE == FIND_COUNT ? 1ull : (u64)exp2(45.0 - ((double)bin + 0.8) / 64.0);
    if (base + held <= (u64)SM_CAP * least) {
      const float s2 = w.no_less(((float)bin + 0.75f) * (1.f / 64.f));
      listed = gather(
          c, row, [&](unsigned bits) { return __uint_as_float(bits) >= s2; },
          [&](unsigned bits, int) {
            double r;
            return w.rough(bits) <= SM_RANGE && w.bin(w.split(w.below(bits), r)) <= bin;
          });
      return 0ull;
    }
  }
  target -= base;
  // bin b has the x that round to 2 b / 128 or (2 b + 1) / 128; beyond SM_RANGE are those that FP32 says so of, off by
  // less than 2^-18
  const float s0 = bin == SM_TAIL ? -INFINITY : w.no_less(((float)bin + 0.75f) * (1.f / 64.f));
  const float s1 = w.no_more(bin == SM_TAIL ? SM_RANGE : ((float)bin - 0.25f) * (1.f / 64.f));
  u64 mn = ~0ull, mx = 0ull, lo = 0ull, hi = ~0ull;
  auto take = [&](unsigned bits, int id, u64& pr) {   // a candidate within the cut and [lo, hi]
    const unsigned key = order_key(bits);
    pr = pair_of(key, id);
    return is_candidate(key) && pr >= cut && pr >= lo && pr <= hi;
  };
  auto span = [&](u64 pr) {
    mn = pr < mn ? pr : mn;
    mx = pr > mx ? pr : mx;
    return true;
  };
  unsigned n = gather(
      c, row,
      [&](unsigned bits) { return __uint_as_float(bits) >= s0 && __uint_as_float(bits) <= s1; },
      [&](unsigned bits, int id) {
        const bool tail = !(w.rough(bits) <= SM_RANGE);
        u64 pr;
        double r;
        if (bin == SM_TAIL ? !tail : tail || w.bin(w.split(w.below(bits), r)) != bin) return false;
        return take(bits, id, pr) && span(pr);
      });
  bool sure = bin != SM_TAIL;            // whether the bin is known to hold the cut
  bool whole = true;                     // whether it holds all candidates of a key, or none
  for (int pass = 0; pass < 10; ++pass) {
    if (n <= SM_CAP) {
      const u64 r = rank_candidates(c, n, MODE, target, w);
      return r ? r : cut;
    }
    mx = warp_max64(mx);
    mn = ~warp_max64(~mn);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) {
      sh->wred[threadIdx.x >> 5] = mx;
      sh->wred2[threadIdx.x >> 5] = mn;
    }
    __syncthreads();
    for (int i = 0; i < SM_WARPS; ++i) {
      mx = sh->wred[i] > mx ? sh->wred[i] : mx;
      mn = sh->wred2[i] < mn ? sh->wred2[i] : mn;
    }
    const int ph = c.exchange(Sel{mx, mn});
    for (int r = 0; r < c.S; ++r) {
      mx = sh->xch[ph][r].a > mx ? sh->xch[ph][r].a : mx;
      mn = sh->xch[ph][r].b < mn ? sh->xch[ph][r].b : mn;
    }
    const unsigned k0 = (unsigned)(mn >> 32), k1 = (unsigned)(mx >> 32);
    int sh_bits;
    if (k0 == k1 && sure && whole && k0 != cut_key) {
      // equal logits: the first ones by id are kept
      const u64 each = MODE == FIND_COUNT ? 1ull : w.weight_of_key(k0);
      const u64 pr = nth_equal(c, row, k0, target / each);
      c.phase ^= 1;                      // it exchanged once
      return pr;
    }
    if (k0 != k1 && whole) {             // by keys, then (rarely) by ids
      lo = pair_of(k0, 0xffffffffu);
      hi = pair_of(k1, 0u);
      sh_bits = 32 + max(0, 21 - __clz((int)(k1 - k0)));   // (k1 - k0) >> (sh_bits - 32) < 2048
    } else {
      lo = mn;
      hi = mx;
      sh_bits = max(0, 53 - __clzll((long long)(hi - lo)));
      whole = false;
    }
    clear_hist(sh);
    auto near_span = [&](unsigned bits_e) {
      const unsigned key = order_key(bits_e);
      return key >= (unsigned)(lo >> 32) && key <= (unsigned)(hi >> 32);
    };
    row.each([&](const unsigned (&x)[8], int id) {
      unsigned mask = 0u;
#pragma unroll
      for (int e = 0; e < 8; ++e) mask |= near_span(x[e]) ? 1u << e : 0u;
      for (; mask; mask &= mask - 1) {
        const int e = __ffs((int)mask) - 1;
        const unsigned xe = nth_of(x, e);
        u64 pr;
        if (!take(xe, id + e, pr)) continue;
        const int at = (int)((hi - pr) >> sh_bits);
        if (MODE == FIND_COUNT)
          atomicAdd(&sh->hist[0][at], 1u);
        else
          add_mass(sh, at, w.weight_of(xe));
      }
      return true;
    });
    bin = locate(c, MODE, 0.f, 0ull, target, base, held, total);
    if (bin < 0) return cut;             // everything is within the target
    sure = true;
    target -= base;
    mn = ~0ull;
    mx = 0ull;
    n = gather(
        c, row, near_span, [&](unsigned bits_e, int id) {
          u64 pr;
          return take(bits_e, id, pr) && (int)((hi - pr) >> sh_bits) == bin && span(pr);
        });
  }
  return cut;                            // not reached: a pass leaves 1/2048 of the range of keys, then of ids
}

// Everything that is left where the row's first candidates in the order are in the list (n of them): ranks, the three
// cuts and the pick.  `mass_limit`: what top-p allows before an element; with top_k it is worked out here.  Every CTA
// does the same; the first one writes.
__device__ __noinline__ void finish_list(Cluster c, const Weigher w, unsigned n, int top_k, float top_p, u64 mass_limit,
                                         double x_max, float u, int row_i, int* ids, int* kept, float* prob) {
  SampleShared* sh = c.sh;
  const u64* cand = sh->cand;
  const int tid = threadIdx.x;
  u64 mine = 0ull, own = 0ull;
  bool in = tid < (int)n;
  __syncthreads();
  if (in) {
    mine = cand[tid];
    own = w.weight_of_key((unsigned)(mine >> 32));
    sh->cand_w[tid] = own;
  }
  __syncthreads();
  unsigned rank = 0u;
  u64 before = 0ull;
  if (in) {
#pragma unroll 8
    for (unsigned j = 0; j < n; ++j) {
      const bool first = cand[j] > mine;
      rank += first;
      before += first ? sh->cand_w[j] : 0ull;
    }
  }
  auto total_of = [&](u64 v, unsigned k, unsigned& count) -> u64 {   // sums of v and k over the threads
    const Sums t = block_sums(sh, warp_sum64(v), __reduce_add_sync(0xffffffffu, k));
    count = (unsigned)t.b;
    return t.a;
  };
  unsigned count;
  if (top_k > 0) {
    in = in && rank < (unsigned)top_k;
    const u64 mass = total_of(in ? own : 0ull, 0u, count);
    mass_limit = part_of(top_p, mass);
  }
  if (top_p < 1.f) in = in && before <= mass_limit;
  const unsigned bits = __float_as_uint(key_value((unsigned)(mine >> 32)));
  if (x_max != INFINITY) {
    const float y = w.rough(bits);
    in = in && (y <= SM_RANGE ? w.below(bits) * w.c : (double)y * 128.0) <= x_max;
  }
  const u64 total = total_of(in ? own : 0ull, in, count);
  if (tid < (int)n) sh->cand_w[tid] = in ? own : 0ull;
  __syncthreads();
  if (c.rank == 0 && in) {
    const u64 target = part_of(u, total);
    const unsigned id = 0xffffffffu - (unsigned)mine;
    u64 at = 0ull;                       // mass of the kept ids below this one
#pragma unroll 8
    for (unsigned j = 0; j < n; ++j) at += 0xffffffffu - (unsigned)cand[j] < id ? sh->cand_w[j] : 0ull;
    if (at <= target && target < at + own) {
      ids[row_i] = (int)id;
      if (kept) kept[row_i] = (int)count;
      if (prob) prob[row_i] = (float)((double)own / (double)total);
    }
  }
  c.sync();                              // no CTA leaves while a peer may still read or write its shared memory
}

template <bool F32>
__global__ void __launch_bounds__(SM_THREADS, 2) sample_kernel(
    const void* logits, long long ld, int V, int lim, int part, int stop_free, UtttSampling opt, const float* u,
    long long u_ld, const int* u_index, int u_len, int* ids, int* kept, float* prob) {
  extern __shared__ __align__(16) uint8_t smem[];
  SampleShared* sh = reinterpret_cast<SampleShared*>(smem);
  Cluster c{cg::this_cluster(), sh, (int)blockIdx.x, (int)gridDim.x, 0, 0};
  const int row_i = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < 2) sh->n_found[tid] = 0u;
  c.arrive();                            // peers write here only once every CTA of the cluster has started
  double pow2[SM_STEPS * 16 / SM_THREADS];   // on their way during the first walk
#pragma unroll
  for (int k = 0; k < SM_STEPS * 16 / SM_THREADS; ++k) pow2[k] = kPow2[(k * SM_THREADS + tid) >> 4];
  pdl_wait();
  pdl_trigger();
  // ---- settings of the row
  float T = opt.temperature ? opt.temperature[row_i] : opt.temperature_all;
  const int top_k = opt.top_k ? opt.top_k[row_i] : opt.top_k_all;
  const float top_p = opt.top_p ? opt.top_p[row_i] : opt.top_p_all;
  const float min_p = opt.min_p ? opt.min_p[row_i] : opt.min_p_all;
  float uv = u[(size_t)row_i * u_ld + (u_index ? min(max(u_index[row_i], 0), u_len - 1) : 0)];
  // ---- the warp's piece of the row (`part` 8-logit vectors per CTA)
  Row<F32> row;
  row.src = reinterpret_cast<const char*>(logits) + (size_t)row_i * ld * (F32 ? 4 : 2);
  row.vec = (reinterpret_cast<uintptr_t>(row.src) & 15u) == 0;
  row.V = V;
  row.has_inf = row.kept = false;
  row.lim = lim;
  row.stop_free = stop_free;
  row.ring = sh->ring[warp];
  const int end = min((c.rank + 1) * part, (lim + 7) / 8), per = ((part + SM_WARPS - 1) / SM_WARPS + 31) & ~31;
  row.v0 = min(end, c.rank * part + warp * per);
  row.v1 = min(end, row.v0 + per);
  float top = -INFINITY;
  row.each([&](const unsigned (&x)[8], int) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) top = max_exact(top, __uint_as_float(x[e]), __uint_as_float(x[e + 1]));
    return true;
  });
  row.kept = row.v1 - row.v0 <= 32 * (F32 ? SM_RING / 2 : SM_RING);
  unsigned mkey = __reduce_max_sync(0xffffffffu, order_key(__float_as_uint(top)));
  if (lane == 0) sh->wred[warp] = mkey;
#pragma unroll
  for (int k = 0; k < SM_STEPS * 16 / SM_THREADS; ++k) sh->tab[k * SM_THREADS + tid] = pow2[k];
  __syncthreads();
  mkey = __reduce_max_sync(0xffffffffu, (unsigned)sh->wred[lane & (SM_WARPS - 1)]);
  c.wait();
  const int ph = c.exchange(Sel{mkey, 0ull});
  mkey = __reduce_max_sync(0xffffffffu, lane < c.S ? (unsigned)sh->xch[ph][lane].a : 0u);
  if (!is_candidate(mkey)) {   // nothing to choose from: an allowed id, as the greedy pick gives
    if (c.rank == 0 && tid == 0) {
      ids[row_i] = (stop_free ? 6 : 2) % lim;
      if (kept) kept[row_i] = 0;
      if (prob) prob[row_i] = 0.f;
    }
    c.sync();                            // no CTA leaves while a peer may still write to it
    return;
  }
  const bool greedy = !(T > SM_GREEDY_T) || top_k == 1;
  Weigher w;
  row.has_inf = mkey == kInfKey;
  if (greedy || row.has_inf) T = 1.f;    // (whatever the temperature, only the infinities have weight)
  const float top_logit = row.has_inf ? kMaxFinite : key_value(mkey);
  w.m = (double)top_logit;
  w.c = 128.0 * 1.4426950408889634074 / (double)T;
  w.scale = T > 1e30f ? 0x1p-100f : 0.5f;
  w.ms = top_logit * w.scale;
  w.cs = (float)(w.c / 128.0 / (double)w.scale);
  w.tab = sh->tab + (lane & 15);
  const double x_max = min_p > 0.f ? -128.0 * log2((double)fminf(min_p, 1.f)) : INFINITY;   // of 128 x
  uv = fminf(uv, 0.99999994f);           // the largest number below 1
  u64 cut = 0ull;
  if (greedy) {
    cut = nth_equal(c, row, order_key(__float_as_uint(top_logit)), 0ull);
    c.phase ^= 1;                        // it exchanged once
  } else {
    unsigned eligible = (unsigned)lim, listed = 0u;
    u64 target = (u64)max(top_k - 1, 0);
    int k_left = 0;                      // what is left for the list to apply
    if (top_k > 0 && top_k < lim) {
      cut = find_cut<FIND_COUNT>(c, row, w, target, 0.f, cut, eligible, listed);
      eligible = (unsigned)top_k;
      k_left = top_k;
    }
    if (listed == 0u && top_p < 1.f) {
      target = 0ull;                     // (stays 0 for top_p <= 0: the first element alone)
      cut = find_cut<FIND_MASS>(c, row, w, target, top_p, cut, eligible, listed);
      k_left = 0;
    }
    if (listed != 0u) {                  // the same in every CTA
      finish_list(c, w, listed, k_left, top_p, target, x_max, uv, row_i, ids, kept, prob);
      return;
    }
  }
  // ---- kept mass per warp
  // The cut is told by the logits themselves, and among equal ones by id; min-p by x, after a quick test.  (A compare
  // takes subnormal numbers for zero: they come out equal at most, and the keys decide.)
  const bool any_cut = cut != 0ull, any_min = x_max != INFINITY;
  const float s_cut = any_cut ? key_value((unsigned)(cut >> 32)) : -INFINITY;
  const float s_low = any_min ? max_exact(s_cut, w.no_less((float)(x_max / 128.0)), -INFINITY) : s_cut;
  // whether an element is above the cut (and perhaps within min-p)
  auto in_cut = [&](unsigned bits, int id) -> bool {
    const float s = __uint_as_float(bits);
    if (s > s_low) return true;
    if (s != s_low) return false;
    const unsigned key = order_key(bits);
    return is_candidate(key) && pair_of(key, id) >= cut;
  };
  // whether such an element is kept, and its weight (a whole number, as a double)
  auto weigh = [&](unsigned bits, double& wt) -> bool {
    const float y = w.rough(bits);
    if (y <= SM_RANGE) {
      const double d = w.below(bits);
      if (any_min && d * w.c > x_max) return false;
      double r;
      const int k = w.split(d, r);
      wt = w.weight52(k, r) - 4503599627370496.0;
      return true;
    }
    if (any_min && (double)y * 128.0 > x_max) return false;   // (min_p below 2^-24)
    wt = (double)w.tail_weight(y);
    return true;
  };
  double sum = 0.0;                      // at most 2^8 weights of 2^45 (SM_MAX_VECS): exact
  unsigned count = 0u;
  auto add = [&](unsigned bits) {
    double wt;
    if (weigh(bits, wt)) {
      sum += wt;
      ++count;
    }
  };
  if (any_cut || any_min) {
    // What is above the cut goes through a list of the warp's own, so that 32 at a time are weighed whichever lanes
    // they came from (the histogram's place is free by now).
    unsigned* const list = &sh->hist[0][0] + warp * (3 * SM_BINS / SM_WARPS);
    static_assert(3 * SM_BINS / SM_WARPS >= 31 + 8 * 32);
    int n = 0;
    row.each([&](const unsigned (&x)[8], int id) {
      unsigned mask = 0u;
#pragma unroll
      for (int e = 0; e < 8; ++e) mask |= in_cut(x[e], id + e) ? 1u << e : 0u;
      const int own = __popc(mask);
      int inc = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += t;
      }
      unsigned* to = list + n + inc - own;
      n += __shfl_sync(0xffffffffu, inc, 31);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (mask >> e & 1u) *to++ = x[e];
      __syncwarp();
      while (n >= 32) {
        n -= 32;
        add(list[n + lane]);
      }
      __syncwarp();
      return true;
    });
    if (lane < n) add(list[lane]);
  } else {
    row.each([&](const unsigned (&x)[8], int id) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (in_cut(x[e], id + e)) add(x[e]);
      return true;
    });
  }
  u64 mass = __double2ull_rn(sum);
  mass = warp_sum64(mass);
  count = __reduce_add_sync(0xffffffffu, count);
  const Sums in = block_sums(sh, mass, count), over = c.sums(c.exchange(Sel{in.a, in.b}));
  const u64 total = over.a, n_kept = over.b, all_below = over.a_below, all = in.a, below = all_below + in.a_below;
  const u64 target = part_of(uv, total);
  // The CTA that holds the pick weighs that warp's piece again, each warp a tile of 32 vectors at a time.
  if (below <= target && target < below + mass) {   // one warp of the cluster
    if (lane == 0) {
      sh->res_bin = warp;
      sh->res_base = below;
    }
  } else if (tid == 0 && !(all_below <= target && target < all_below + all)) {
    sh->res_bin = -1;
  }
  __syncthreads();
  const int owner = sh->res_bin;
  const int p0 = min(end, c.rank * part + max(owner, 0) * per), p1 = owner >= 0 ? min(end, p0 + per) : p0;
  u64 piece = sh->res_base;              // mass before the tiles
  row.kept = false;
  for (int v0 = p0; v0 < p1 && piece <= target; v0 += SM_THREADS) {   // the same for the whole CTA
    row.v0 = min(p1, v0 + warp * 32);
    row.v1 = min(p1, row.v0 + 32);
    u64 wt[8], own = 0ull;
    int id0 = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) wt[e] = 0ull;
    row.each([&](const unsigned (&x)[8], int id) {   // one vector a lane
      id0 = id;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        double v;
        wt[e] = in_cut(x[e], id + e) && weigh(x[e], v) ? mantissa(v + 4503599627370496.0) : 0ull;
        own += wt[e];
      }
      return true;
    });
    u64 inc = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 t = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += t;
    }
    const Sums tiles = block_sums(sh, __shfl_sync(0xffffffffu, inc, 31), 0ull);
    u64 run = piece + inc - own + tiles.a_below;
    piece += tiles.a;
    if (run <= target && target < run + own) {       // one lane
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (run <= target && target < run + wt[e]) {
          ids[row_i] = id0 + e;
          if (kept) kept[row_i] = (int)n_kept;
          if (prob) prob[row_i] = (float)((double)wt[e] / (double)total);
        }
        run += wt[e];
      }
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
  // A row is split over a cluster of S while the rows alone leave SMs idle (two CTAs fit an SM; at least 2048 logits per
  // CTA), and where a CTA's part would be too large for the histogram's limbs (ids 0, 1 and 3 are no candidates) or for
  // the lanes' sums.
  // At top-p 0.95, S = 1 / 2 / 4 / 8, launches one by one: one row of 32000 46 / 40 / 34 / 32 us, 64 rows 53 / 42 / 42 /
  // 63, 333 rows of 8003 53 / 73 / 124 / 250, 256 rows of 131072 199 / 222 / 266 / 362.
  const int nvec = (lim + 7) / 8;
  int S = 1;
  while (S < SM_MAX_CTAS && ((S == 1 ? lim - 3 : (nvec + S - 1) / S * 8) > SM_MAX_PART ||
                             (nvec + S - 1) / S > SM_MAX_VECS ||
                             ((long long)rows * 2 * S <= 2 * num_sms() && lim / (2 * S) >= 2048)))
    S *= 2;
  const int part = (nvec + S - 1) / S;
  auto kernel = logits_f32 ? sample_kernel<true> : sample_kernel<false>;
  static DeviceOnce attr;
  UTTT_TRY(run_once_per_device(attr, [] {
    UTTT_TRY(cuda_status(cudaFuncSetAttribute(sample_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                              (int)sizeof(SampleShared))));
    return cuda_status(cudaFuncSetAttribute(sample_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            (int)sizeof(SampleShared)));
  }));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(S, rows);
  cfg.blockDim = dim3(SM_THREADS);
  cfg.dynamicSmemBytes = sizeof(SampleShared);
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = S;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  at[1] = pdl_attribute();
  cfg.attrs = at;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, kernel, logits, ld, V, lim, part, stop_free, *opt, u, u_ld, u_index, u_len, ids, kept,
                         prob) != cudaSuccess)
    return launch_status();
  return launch_status();
}
