// Drafted tokens arranged as a tree: attention of all nodes of a tree over a
// persona's KV ring, and the path of the tree that the picks accept.
//
// Attention.  Row b of the batch holds up to N nodes; node i has parent
// parents[b][i] < i, depth d_i (roots: 0) and absolute position pos[b] + d_i.  It
// sees the ring's positions in (pos + d_i - W, pos) and the nodes on its own
// path (itself and its ancestors) that are less than W deep above it, so every
// path of the tree gets what uttt_attn_decode would give it token by token:
// o_i = sum_j softmax_j(q_i . k_j / sqrt(hd)) v_j.  The ring is only read: the
// nodes' RoPE'd keys and values go to k_tree / v_tree, and uttt_kv_ring_commit
// copies an accepted path into the ring.  RoPE rounds as the decode kernel does.
//
// Kernels.  The rep query heads of a KV head and the nodes stack into the rows of
// one matrix product (row = node * rep + head), so a ring is read once for all of
// them.  One CTA takes up to 128 rows and streams its share of the keys through
// shared memory in 64-key tiles; the drafted keys, RoPE'd on the way, are the
// first one.  Per row it keeps the running maximum and sum of the softmax and the
// unnormalised output.  With few rows in the batch a cluster of S CTAs splits the
// keys and joins its partials in distributed shared memory.
//   head dim 64, 128   attn_tree_tc_kernel: tcgen05, S and O in TMEM, TMA tiles;
//   head dim 32        attn_tree_kernel: mma.sync (16 x 8 x 16), cp.async tiles
//                      (a row is half of the 128-byte swizzle the others use).
// mma.sync for few rows of the larger heads was measured and dropped: 64 rows of
// 8 nodes at the 1.58B heads (32 rows a CTA) 40.4 us against 31.6 us here, 4 nodes
// (16 rows) 31.0 against 31.6, 32 rows of 5 nodes at 12/4 heads 14.2 against 12.8.
// The probabilities enter the second product as two BF16 parts, P_hi = bf16(P) and
// P_lo = bf16(P - P_hi) (about 16 significant bits, as the prefill kernel does);
// scores, statistics and sums are FP32.
//
// What bounds it (1.58B heads unless said).  64 rows of 1 to 16 nodes over window
// 512: 30.4 us, of which 59 rows in one wave take 22.5; of a CTA's 28000 cycles 8500
// are the nodes' paths, loads and RoPE before the first tile and 2400 the output,
// between them the rings stream at the HBM rate (77 MB).  8 rows of 31 nodes over
// window 8192, one KV head: 32.6 us.  One of its CTAs ends after 43900 cycles (22 us):
// 9300 before the first tile, 24000 in 16 tiles (1500 each: the softmax between two
// products on the tensor cores, its powers alone 512) and 9700 for the cluster's join;
// the rest is SMs that hold two such CTAs while others hold none (the tensor pipe is
// busy 57 % on the busiest SM, 25 % on average).  One row of 5 nodes: 13 us, the
// host's side of the call (9 in a captured graph).  Head dim 32: 28 us for the 64
// rows, 46 for the 8 over window 8192.
#include <cooperative_groups.h>

#include "common.cuh"
#include "host_util.cuh"

namespace cg = cooperative_groups;

namespace uttt {
namespace {

constexpr int TR_MAX_N = 64;
constexpr int TR_MAX_REP = 8;

__device__ __forceinline__ float bfr(float x) { return __bfloat162float(__float2bfloat16(x)); }

constexpr int TR_KT = 64;                // keys per tile (and the most nodes of a tree)
constexpr int TR_HD = 32;                // head dim of the mma.sync kernel ...
constexpr int TR_NS = 3;                 // ... and its tiles in flight

typedef unsigned long long u64;

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// byte offset of 16-byte chunk c of row r in a tile of 32-element rows; the XOR spreads the 8 rows of an
// ldmatrix over all banks
__device__ __forceinline__ uint32_t tile_off(int r, int c) { return (uint32_t)(r * 64 + ((c ^ ((r >> 1) & 3)) << 4)); }

__device__ __forceinline__ bool has_nonfinite(uint32_t v) {   // either BF16 half
  return (v & 0x7f80u) == 0x7f80u || (v & 0x7f800000u) == 0x7f800000u;
}
__device__ __forceinline__ uint32_t finite_only(uint32_t v) {
  if ((v & 0x7f80u) == 0x7f80u) v &= 0xffff0000u;
  if ((v & 0x7f800000u) == 0x7f800000u) v &= 0x0000ffffu;
  return v;
}

struct TreeArgs {
  const __nv_bfloat16* qkv;
  const int *parents, *n_nodes, *pos, *slot;
  const __nv_bfloat16 *kring, *vring;
  const float *cos_t, *sin_t;
  __nv_bfloat16 *ktree, *vtree, *out;
  int qkv_ld, N, n_kv, rep, W, n_slots, n_pos, out_ld;
  float scale_log2;                      // log2(e) / sqrt(hd)
  int vec_in, vec_out;                   // whether rows of qkv (with the tables) and of out start on 16 bytes
  int b0;                                // the first row of the launch
  int joins;                             // whether the launch is the rest of the one before it
  int* status;                           // receives UTTT_ERR_TIMEOUT if a wait expires (or null)
  uint32_t max_polls;                    // of a CTA's loads for a free slot
};

// bits lo .. lo + len - 1, as far as they lie in 0 .. 63
__device__ __forceinline__ u64 bit_range(int lo, int len) {
  const int a = max(lo, 0), b = min(lo + len, 64);
  return b > a ? (~0ull >> (64 - (b - a))) << a : 0ull;
}
// Of the ring places j0 .. j0 + 63: those that a node `depth` deep does not see any more, the depth + 1 places
// behind `next`, the oldest one (place j holds the position (j - next) mod W behind the oldest).
__device__ __forceinline__ u64 hidden_places(int j0, int next, int W, int depth) {
  return bit_range(next - j0, depth + 1) | bit_range(next - W - j0, depth + 1);
}

// what other SMs' completed writes hold is seen by the loads and the asynchronous copies that follow
__device__ __forceinline__ void fence_device() {
  asm volatile("fence.acq_rel.gpu;" ::: "memory");
  asm volatile("fence.proxy.async.global;" ::: "memory");
}

__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// 8 elements of a row of qkv
template <bool VEC>
__device__ __forceinline__ uint4 load8(const __nv_bfloat16* p) {
  if (VEC) return *reinterpret_cast<const uint4*>(p);
  const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
  return make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16, h[4] | (uint32_t)h[5] << 16,
                    h[6] | (uint32_t)h[7] << 16);
}
// 8 table values, rounded to BF16 as apply_rope does
template <bool VEC>
__device__ __forceinline__ void load_trig(uint32_t (&t)[4], const float* p) {
  if (VEC) {
    const float4 x = reinterpret_cast<const float4*>(p)[0], y = reinterpret_cast<const float4*>(p)[1];
    t[0] = pack_bf16x2(x.x, x.y), t[1] = pack_bf16x2(x.z, x.w);
    t[2] = pack_bf16x2(y.x, y.y), t[3] = pack_bf16x2(y.z, y.w);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = pack_bf16x2(p[2 * i], p[2 * i + 1]);
  }
}
__device__ __forceinline__ __nv_bfloat162& as_bf162(uint32_t& v) { return reinterpret_cast<__nv_bfloat162&>(v); }

// Table values of 8 elements of the first half of a head vector and of their partners in the second.
struct Trig {
  uint32_t cl[4], ch[4], sl[4], sh[4];
  template <bool VEC>
  __device__ __forceinline__ void load(const float* cosr, const float* sinr, int i0, int half) {
    load_trig<VEC>(cl, cosr + i0);
    load_trig<VEC>(ch, cosr + i0 + half);
    load_trig<VEC>(sl, sinr + i0);
    load_trig<VEC>(sh, sinr + i0 + half);
  }
  // rotate-half RoPE, every product and the sum rounded to BF16 as apply_rope (model/uttt_layer.py:946-958): BF16
  // arithmetic rounds each of them once (a product of two BF16 values is exact in FP32, and so is every sum that
  // is near a rounding border)
  __device__ __forceinline__ void rotate(uint4& lo, uint4& hi) {
    uint32_t* l = reinterpret_cast<uint32_t*>(&lo);
    uint32_t* h = reinterpret_cast<uint32_t*>(&hi);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const __nv_bfloat162 xl = as_bf162(l[k]), xh = as_bf162(h[k]);
      as_bf162(l[k]) = __hsub2_rn(__hmul2_rn(xl, as_bf162(cl[k])), __hmul2_rn(xh, as_bf162(sl[k])));
      as_bf162(h[k]) = __hadd2_rn(__hmul2_rn(xh, as_bf162(ch[k])), __hmul2_rn(xl, as_bf162(sh[k])));
    }
  }
};

// RoPE of the CTA's query rows row0 .. row0 + n_rows - 1 and, with `tree`, of the nodes' keys, and the nodes' values.
// A thread takes 8 elements and their partners of every head of one node, so the table values are read once and all
// of a node's loads are in flight together.  put_q / put_k / put_v(r, c, v) take 16-byte chunk c of row or node r;
// `keep` marks the CTA that writes k_tree and v_tree.  Non-finite values are left out of put_v and their nodes
// marked in *bad: 0 * NaN would let a key's value reach rows that do not see it; they are added at the end to the
// rows that do.
template <int HD, bool VEC, class Depth, class PutQ, class PutK, class PutV>
__device__ __forceinline__ void rope_nodes_as(int tid, int threads, int n, int b, int g, int p0, int row0, int n_rows,
                                              bool tree, const TreeArgs& a, u64* bad, Depth depth, PutQ put_q,
                                              PutK put_k, PutV put_v) {
  constexpr int HC = HD / 16, CH = HD / 8;
  const __nv_bfloat16* rows = a.qkv + (size_t)b * a.N * a.qkv_ld;
  const int rep = a.rep, nodes = tree ? n : min(n, (row0 + n_rows + rep - 1) / rep);
  const int first = tree ? 0 : row0 / rep;
  const bool keep = tree && row0 == 0;
  for (int i = tid; i < (nodes - first) * HC; i += threads) {
    const int node = first + i / HC, c = i % HC;
    const __nv_bfloat16* x = rows + (size_t)node * a.qkv_ld + c * 8;
    const __nv_bfloat16* xq = x + (size_t)g * rep * HD;
    const __nv_bfloat16* xk = x + (size_t)(a.n_kv * rep + g) * HD;
    const __nv_bfloat16* xv = xk + (size_t)a.n_kv * HD;
    const size_t tr = (size_t)min((long long)p0 + depth(node), (long long)a.n_pos - 1) * HD;
    const int r0 = node * rep - row0;
    uint4 k0, k1, v0, v1;
    if (tree) {
      k0 = load8<VEC>(xk);
      k1 = load8<VEC>(xk + HD / 2);
      v0 = load8<VEC>(xv);
      v1 = load8<VEC>(xv + HD / 2);
    }
    Trig t;
#pragma unroll
    for (int h0 = 0; h0 < TR_MAX_REP; h0 += 4) {
      if (h0 >= rep) break;
      uint4 lo[4], hi[4];
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const int r = r0 + h0 + h;
        if (h0 + h < rep && r >= 0 && r < n_rows) {
          lo[h] = load8<VEC>(xq + (size_t)(h0 + h) * HD);
          hi[h] = load8<VEC>(xq + (size_t)(h0 + h) * HD + HD / 2);
        }
      }
      if (h0 == 0) t.template load<VEC>(a.cos_t + tr, a.sin_t + tr, c * 8, HD / 2);
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const int r = r0 + h0 + h;
        if (h0 + h < rep && r >= 0 && r < n_rows) {
          t.rotate(lo[h], hi[h]);
          put_q(r, c, lo[h]);
          put_q(r, c + HC, hi[h]);
        }
      }
    }
    if (tree) {
      t.rotate(k0, k1);
      put_k(node, c, k0);
      put_k(node, c + HC, k1);
      if (keep) {
        const size_t o = (((size_t)b * a.n_kv + g) * a.N + node) * HD + c * 8;
        *reinterpret_cast<uint4*>(a.ktree + o) = k0;
        *reinterpret_cast<uint4*>(a.ktree + o + HD / 2) = k1;
        *reinterpret_cast<uint4*>(a.vtree + o) = v0;
        *reinterpret_cast<uint4*>(a.vtree + o + HD / 2) = v1;
      }
      if (has_nonfinite(v0.x) || has_nonfinite(v0.y) || has_nonfinite(v0.z) || has_nonfinite(v0.w) ||
          has_nonfinite(v1.x) || has_nonfinite(v1.y) || has_nonfinite(v1.z) || has_nonfinite(v1.w)) {
        v0 = make_uint4(finite_only(v0.x), finite_only(v0.y), finite_only(v0.z), finite_only(v0.w));
        v1 = make_uint4(finite_only(v1.x), finite_only(v1.y), finite_only(v1.z), finite_only(v1.w));
        atomicOr(bad, 1ull << node);
      }
      put_v(node, c, v0);
      put_v(node, c + HC, v1);
    }
  }
  // zeros behind the last query row and the last node
  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (int i = tid + max(0, min(n_rows, n * rep - row0)) * CH; i < n_rows * CH; i += threads) put_q(i / CH, i % CH, zero);
  if (tree)
    for (int i = tid + n * CH; i < TR_KT * CH; i += threads) {
      put_k(i / CH, i % CH, zero);
      put_v(i / CH, i % CH, zero);
    }
}
template <int HD, class... F>
__device__ __forceinline__ void rope_nodes(int tid, int threads, int n, int b, int g, int p0, int row0, int n_rows,
                                           bool tree, const TreeArgs& a, u64* bad, F... f) {
  if (a.vec_in)
    rope_nodes_as<HD, true>(tid, threads, n, b, g, p0, row0, n_rows, tree, a, bad, f...);
  else
    rope_nodes_as<HD, false>(tid, threads, n, b, g, p0, row0, n_rows, tree, a, bad, f...);
}

// The same for the values of the keys `keys` of a ring tile in shared memory, at(r, c) being chunk c of key r.
template <int HD, class At>
__device__ __forceinline__ void finite_values(int tid, int threads, u64 keys, u64* bad, At at) {
  constexpr int CH = HD / 8;
  if (!keys) return;
  const int r0 = __ffsll((long long)keys) - 1, r1 = 63 - __clzll((long long)keys);
  for (int i = tid; i < (r1 - r0 + 1) * CH; i += threads) {
    const int r = r0 + i / CH;
    if (!((keys >> r) & 1ull)) continue;
    uint4* p = at(r, i % CH);
    const uint4 v = *p;
    if (has_nonfinite(v.x) || has_nonfinite(v.y) || has_nonfinite(v.z) || has_nonfinite(v.w)) {
      *p = make_uint4(finite_only(v.x), finite_only(v.y), finite_only(v.z), finite_only(v.w));
      atomicOr(bad, 1ull << r);
    }
  }
}

// What a CTA reads of qkv and of the tables, on its way to L2 while the nodes' paths are worked out.
template <int HD>
__device__ __forceinline__ void prefetch_nodes(int tid, int threads, int n, int b, int g, int p0, const TreeArgs& a) {
  const char* q = reinterpret_cast<const char*>(a.qkv + (size_t)b * a.N * a.qkv_ld);
  const int qb = a.rep * HD * 2, per = (qb + 127) / 128 + 2 * ((HD * 2 + 127) / 128);   // 128-byte lines per node
  for (int i = tid; i < n * per; i += threads) {
    const int r = i / per, k = i % per, kl = (HD * 2 + 127) / 128, ql = per - 2 * kl;
    const int off = k < ql ? g * qb + k * 128
                           : (a.n_kv * a.rep + g + (k >= ql + kl ? a.n_kv : 0)) * HD * 2 + (k - ql) % kl * 128;
    prefetch_l2(q + (size_t)r * a.qkv_ld * 2 + off);
  }
  // positions p0 .. are the depths'; few trees are deeper than 16
  const int rows = min(min(n, 16), a.n_pos - min(p0, a.n_pos));
  for (int i = tid; i < rows * (HD * 4 / 128) * 2; i += threads) {
    const float* t = (i & 1) ? a.sin_t : a.cos_t;
    prefetch_l2(reinterpret_cast<const char*>(t + (size_t)p0 * HD) + (i >> 1) * 128);
  }
}

// The partials of a row, joined by CTA r % S of the cluster: every CTA sends its maximum, sum and unnormalised output
// there (remote stores, nobody waits for them one by one), at [sender][r / S].
struct Joiner {
  float* o;                              // [S][rows / S][old]
  float (*ml)[2];                        // [S][rows / S]
  int S, per, old;                       // per: rows per CTA
  __device__ __forceinline__ void send_ml(cg::cluster_group& cl, int z, int r, float m, float l) const {
    float* p = cl.map_shared_rank(&ml[z * per + r / S][0], r % S);
    p[0] = m;
    p[1] = l;
  }
  __device__ __forceinline__ float4* row(cg::cluster_group& cl, int z, int r) const {
    return reinterpret_cast<float4*>(cl.map_shared_rank(o + (size_t)(z * per + r / S) * old, r % S));
  }
  // columns c8 .. c8 + 7 of this CTA's row number q (row q * S + rank); returns the sum
  __device__ __forceinline__ float join(int q, int c8, float (&v)[8]) const {
    float M = -INFINITY, L = 0.f;
    for (int k = 0; k < S; ++k) M = fmaxf(M, ml[k * per + q][0]);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    for (int k = 0; k < S; ++k) {
      const float mk = ml[k * per + q][0];
      if (mk == -INFINITY) continue;     // a CTA whose keys this row does not see
      const float f = exp2f(mk - M);
      L += f * ml[k * per + q][1];
      const float4* p = reinterpret_cast<const float4*>(o + (size_t)(k * per + q) * old + c8);
      const float4 x = p[0], y = p[1];
      v[0] += f * x.x, v[1] += f * x.y, v[2] += f * x.z, v[3] += f * x.w;
      v[4] += f * y.x, v[5] += f * y.y, v[6] += f * y.z, v[7] += f * y.w;
    }
    return L;
  }
};

// 8 columns of a row of out
__device__ __forceinline__ void store_out(const TreeArgs& a, int b, int g, int row, int c8, int hd, const float (&v)[8],
                                          float inv) {
  const int node = row / a.rep, h = g * a.rep + row % a.rep;
  __nv_bfloat16* dst = a.out + ((size_t)b * a.N + node) * a.out_ld + (size_t)h * hd + c8;
  if (a.vec_out) {
    *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16x2(v[0] * inv, v[1] * inv), pack_bf16x2(v[2] * inv, v[3] * inv),
                                                pack_bf16x2(v[4] * inv, v[5] * inv), pack_bf16x2(v[6] * inv, v[7] * inv));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) dst[e] = __float2bfloat16(v[e] * inv);
  }
}

template <int WM>
__host__ __device__ constexpr int tree_threads() { return 32 * (WM < 4 ? 4 : WM); }
// the tiles; at the end the warps' partials and, behind them, the rows that the cluster sends
template <int WM>
constexpr int tree_smem() {
  constexpr int tiles = TR_NS * 2 * TR_KT * TR_HD * 2, ends = (tree_threads<WM>() / 32 + WM) * 16 * (TR_HD + 4) * 4;
  return tiles > ends ? tiles : ends;
}

// CTAs that share a row's keys.  A CTA takes about as long as `head` tiles before and after its own tiles (node
// paths, RoPE, output), a cluster `join` more; S minimises the waves of CTAs times that.  (Clusters of 16, for long
// windows: 44.5 us against 32.5 for 8 rows of 31 nodes and window 8192; the GPU does not hold 16 of them at a time.)
inline int tree_split(long long ctas, int tiles, int per_sm, int head, int join) {
  const long long slots = (long long)num_sms() * per_sm;
  int best = 1;
  long long least = 0;
  for (int S = 1; S <= 8 && (S == 1 || tiles >= 2 * S); S *= 2) {
    const long long waves = (ctas * S + slots - 1) / slots;
    const long long cost = waves * (head + (tiles + S - 1) / S + (S > 1 ? join : 0));
    if (S == 1 || cost < least) {
      best = S;
      least = cost;
    }
  }
  return best;
}

// Head dim 32.  WM warps stack along the rows (16 each) and WK along the keys of a tile, so that a few rows still
// use every warp; three tiles are in flight.
// grid (S, n_kv * row blocks, B), cluster (S, 1, 1): CTA z takes tiles [nt * z / S, nt * (z + 1) / S) of the nt
// 64-key tiles: tile 0 holds the drafted keys, tile t > 0 the ring's places 64 (t - 1) ..
template <int WM>
__global__ void __launch_bounds__(tree_threads<WM>()) attn_tree_kernel(const TreeArgs a) {
  constexpr int HD = TR_HD, THREADS = tree_threads<WM>(), NW = THREADS / 32, WK = NW / WM;
  constexpr int RB = 16 * WM;            // rows of the CTA
  constexpr int KW = TR_KT / WK;         // keys of a tile per warp
  constexpr int SUB = KW < 32 ? KW : 32;  // keys between two updates of the running maximum
  constexpr int CH = HD / 8, TILE = TR_KT * HD * 2;
  constexpr int OLD = HD + 4;            // row stride of the partial outputs (floats): rows shift by 4 banks
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ u64 anc_s[2][TR_KT], bad_keys, bad_tree;
  __shared__ int jump_s[2][TR_KT], depth_s[TR_KT], deepest;
  __shared__ float m_s[NW][16], l_s[NW][16], fac_s[WK][RB], cml[2][RB], ml_s[RB][2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, wm = warp % WM, wk = warp / WM;
  const int S = gridDim.x, z = blockIdx.x, b = blockIdx.z;
  const int g = blockIdx.y % a.n_kv, row0 = blockIdx.y / a.n_kv * RB;
  const int N = a.N, rep = a.rep, W = a.W;
  pdl_wait();
  pdl_trigger();
  const int par_i = tid < N ? a.parents[(size_t)b * N + tid] : -1;
  const int n = a.n_nodes ? min(a.n_nodes[b], N) : N;
  const int p0 = a.pos[b], sl = a.slot[b];
  const int rows = n * rep;              // rows of the whole (row, KV head)
  if (row0 >= rows || sl < 0 || sl >= a.n_slots || p0 < 0) return;   // the same in the whole cluster

  // ---- ring tiles on their way first
  const int nvalid = min(p0, W), nt = (nvalid + TR_KT - 1) / TR_KT + 1;
  const int t_lo = (int)((long long)nt * z / S), t_hi = (int)((long long)nt * (z + 1) / S);
  const bool has_tree = t_lo == 0 && t_hi > 0;
  const size_t ring0 = ((size_t)sl * a.n_kv + g) * (size_t)W * HD;
  const __nv_bfloat16* qrows = a.qkv + (size_t)b * N * a.qkv_ld;
  const int v_col = (a.n_kv * (rep + 1) + g) * HD;
  auto load_ring = [&](int t) {
    uint8_t* ks = smem + ((t - t_lo) % TR_NS) * 2 * TILE;
    for (int i = tid; i < TR_KT * CH; i += THREADS) {
      const int r = i / CH, c = i % CH, j = (t - 1) * TR_KT + r;
      const bool ok = j < nvalid;
      const size_t o = ring0 + (size_t)(ok ? j : 0) * HD + c * 8;
      cp_async_16(ks + tile_off(r, c), a.kring + o, ok);
      cp_async_16(ks + TILE + tile_off(r, c), a.vring + o, ok);
    }
  };
#pragma unroll
  for (int i = 0; i < TR_NS - 1; ++i) {
    if (t_lo + i < t_hi && t_lo + i > 0) load_ring(t_lo + i);
    cp_async_commit();
  }
  prefetch_nodes<HD>(tid, THREADS, n, b, g, p0, a);

  // ---- every node's path as a bit mask, by pointer jumping (6 doublings reach 64 ancestors)
  if (tid == 0) {
    bad_tree = 0ull;
    deepest = 0;
  }
  if (tid < TR_KT) {
    anc_s[0][tid] = 1ull << tid;
    jump_s[0][tid] = tid < n && par_i >= 0 && par_i < tid ? par_i : -1;   // anything else makes a root
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 6; ++k) {
    if (tid < TR_KT) {
      const int j = jump_s[k & 1][tid];
      anc_s[(k & 1) ^ 1][tid] = anc_s[k & 1][tid] | (j >= 0 ? anc_s[k & 1][j] : 0ull);
      jump_s[(k & 1) ^ 1][tid] = j >= 0 ? jump_s[k & 1][j] : -1;
    }
    __syncthreads();
  }
  if (tid < TR_KT) {
    u64 m = anc_s[0][tid];
    const int d = __popcll(m) - 1;
    depth_s[tid] = d;
    if (tid < n && d > 0) atomicMax(&deepest, d);
    if (d >= W)                          // ancestors that have left the window
      for (u64 rest = m; rest; rest &= rest - 1) {
        const int j = __ffsll((long long)rest) - 1;
        if (d - (__popcll(anc_s[0][j]) - 1) >= W) m &= ~(1ull << j);
      }
    anc_s[1][tid] = m;
  }
  __syncthreads();

  // ---- RoPE: Q into the last stage (then registers); the drafted keys and values are the first tile
  uint8_t* sQ = smem + (TR_NS - 1) * 2 * TILE;
  rope_nodes<HD>(
      tid, THREADS, n, b, g, p0, row0, RB, has_tree, a, &bad_tree, [&](int node) { return depth_s[node]; },
      [&](int r, int c, uint4 v) { *reinterpret_cast<uint4*>(sQ + tile_off(r, c)) = v; },
      [&](int r, int c, uint4 v) { *reinterpret_cast<uint4*>(smem + tile_off(r, c)) = v; },
      [&](int r, int c, uint4 v) { *reinterpret_cast<uint4*>(smem + TILE + tile_off(r, c)) = v; });
  __syncthreads();
  uint32_t qf[HD / 16][4];
#pragma unroll
  for (int k = 0; k < HD / 16; ++k)
    ldsm4(qf[k], smem_u32(sQ) + tile_off(wm * 16 + (lane & 15), 2 * k + (lane >> 4)));

  // ---- this thread's two rows (lane / 4 and + 8 of its warp's 16)
  int dep[2];
  u64 anc[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int row = row0 + wm * 16 + (lane >> 2) + 8 * e;
    const bool ok = row < rows;
    dep[e] = ok ? depth_s[row / rep] : -1;
    anc[e] = ok ? anc_s[1][row / rep] : ~0ull;
  }
  const int next = p0 % W, max_dep = deepest;   // next: the oldest place
  float o[HD / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < HD / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.f;

  for (int t = t_lo; t < t_hi; ++t) {
    cp_async_wait<TR_NS - 2>();
    __syncthreads();
    if (t + TR_NS - 1 < t_hi) load_ring(t + TR_NS - 1);
    cp_async_commit();
    uint8_t* ks = smem + ((t - t_lo) % TR_NS) * 2 * TILE;
    const uint32_t ka = smem_u32(ks), va = ka + TILE;
    const bool is_tree = t == 0;
    // keys that not every row sees: the tree's, the ring's behind the last valid place and around the window's edge
    const int j0 = (t - 1) * TR_KT;
    const u64 some = is_tree ? ~0ull : hidden_places(j0, next, W, max_dep);
    const bool edge = is_tree || j0 + TR_KT > nvalid || some != 0ull;
    u64 bad = 0ull, seen[2] = {~0ull, ~0ull};
    if (edge) {
      if (is_tree) {
        bad = bad_tree;
        seen[0] = anc[0];
        seen[1] = anc[1];
      } else {
        const u64 valid = bit_range(0, nvalid - j0);
        if (some & valid) {
          if (tid == 0) bad_keys = 0ull;
          __syncthreads();
          finite_values<HD>(tid, THREADS, some & valid, &bad_keys, [&](int r, int c) {
            return reinterpret_cast<uint4*>(ks + TILE + tile_off(r, c));
          });
          __syncthreads();
          bad = bad_keys;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) seen[e] = valid & ~hidden_places(j0, next, W, dep[e]);
      }
    }
#pragma unroll
    for (int sub = 0; sub < KW / SUB; ++sub) {
      const int kb = wk * KW + sub * SUB;
      float s[SUB / 8][4];
#pragma unroll
      for (int i = 0; i < SUB / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i][e] = 0.f;
#pragma unroll
      for (int k = 0; k < HD / 16; ++k)
#pragma unroll
        for (int i = 0; i < SUB / 16; ++i) {
          uint32_t kf[4];
          ldsm4(kf, ka + tile_off(kb + i * 16 + (lane & 7) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1)));
          mma16816(s[2 * i], qf[k], kf[0], kf[1]);
          mma16816(s[2 * i + 1], qf[k], kf[2], kf[3]);
        }
      if (edge) {
        // bits of this thread's columns: i * 8 and i * 8 + 1 after the shift
        const uint32_t v0 = (uint32_t)(seen[0] >> (kb + (lane & 3) * 2)), v1 = (uint32_t)(seen[1] >> (kb + (lane & 3) * 2));
#pragma unroll
        for (int i = 0; i < SUB / 8; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!(((e >> 1) ? v1 : v0) >> (i * 8 + (e & 1)) & 1u)) s[i][e] = -INFINITY;
      }
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < SUB / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[i][e] *= a.scale_log2;
          mx[e >> 1] = fmaxf(mx[e >> 1], s[i][e]);
        }
      float c[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
        mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
        mx[e] = fmaxf(mx[e], m[e]);
        c[e] = mx[e] > m[e] ? exp2f(m[e] - mx[e]) : 1.f;
        m[e] = mx[e];
        l[e] *= c[e];
        if (mx[e] == -INFINITY) mx[e] = 0.f;   // nothing seen yet: every weight below is 0
      }
      if (__any_sync(0xffffffffu, c[0] != 1.f || c[1] != 1.f))
#pragma unroll
        for (int i = 0; i < HD / 8; ++i) {
          o[i][0] *= c[0];
          o[i][1] *= c[0];
          o[i][2] *= c[1];
          o[i][3] *= c[1];
        }
      uint32_t ph[SUB / 16][4], pl[SUB / 16][4];
#pragma unroll
      for (int i = 0; i < SUB / 8; ++i) {
        float q[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          q[e] = exp2f(s[i][e] - mx[e >> 1]);
          l[e >> 1] += q[e];
          lo[e] = q[e] - bfr(q[e]);
        }
        ph[i >> 1][(i & 1) * 2] = pack_bf16x2(q[0], q[1]);
        ph[i >> 1][(i & 1) * 2 + 1] = pack_bf16x2(q[2], q[3]);
        pl[i >> 1][(i & 1) * 2] = pack_bf16x2(lo[0], lo[1]);
        pl[i >> 1][(i & 1) * 2 + 1] = pack_bf16x2(lo[2], lo[3]);
      }
#pragma unroll
      for (int i = 0; i < SUB / 16; ++i)
#pragma unroll
        for (int cc = 0; cc < HD / 16; ++cc) {
          uint32_t vf[4];
          ldsm4_t(vf, va + tile_off(kb + i * 16 + (lane & 15), 2 * cc + (lane >> 4)));
          mma16816(o[2 * cc], ph[i], vf[0], vf[1]);
          mma16816(o[2 * cc + 1], ph[i], vf[2], vf[3]);
          mma16816(o[2 * cc], pl[i], vf[0], vf[1]);
          mma16816(o[2 * cc + 1], pl[i], vf[2], vf[3]);
        }
    }
    for (u64 rest = bad; rest; rest &= rest - 1) {
      const int key = __ffsll((long long)rest) - 1;
      if (key / KW != wk) continue;
      const __nv_bfloat16* v = is_tree ? qrows + (size_t)key * a.qkv_ld + v_col
                                       : a.vring + ring0 + (size_t)(j0 + key) * HD;
#pragma unroll
      for (int i = 0; i < HD / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = __bfloat162float(v[i * 8 + (lane & 3) * 2 + (e & 1)]);
          if ((__float_as_uint(x) & 0x7f800000u) == 0x7f800000u && (seen[e >> 1] >> key & 1ull)) o[i][e] += x;
        }
    }
  }
  cp_async_wait<0>();

  // ---- partials: warps of one row block, then the CTAs of the cluster
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
  }
  __syncthreads();                       // every warp has read its last tile
  float* part = reinterpret_cast<float*>(smem);   // [NW][16][OLD]
  {
    float* po = part + (size_t)warp * 16 * OLD;
    const int r = lane >> 2, cq = (lane & 3) * 2;
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) {
      *reinterpret_cast<float2*>(po + r * OLD + i * 8 + cq) = make_float2(o[i][0], o[i][1]);
      *reinterpret_cast<float2*>(po + (r + 8) * OLD + i * 8 + cq) = make_float2(o[i][2], o[i][3]);
    }
    if ((lane & 3) == 0) {
      m_s[warp][r] = m[0];
      m_s[warp][r + 8] = m[1];
      l_s[warp][r] = l[0];
      l_s[warp][r + 8] = l[1];
    }
  }
  __syncthreads();
  if (tid < RB) {                        // row tid: warps (tid / 16) + k * WM
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int k = 0; k < WK; ++k) M = fmaxf(M, m_s[(tid >> 4) + k * WM][tid & 15]);
#pragma unroll
    for (int k = 0; k < WK; ++k) {
      const float mk = m_s[(tid >> 4) + k * WM][tid & 15];
      const float f = mk == -INFINITY ? 0.f : exp2f(mk - M);
      fac_s[k][tid] = f;
      L += f * l_s[(tid >> 4) + k * WM][tid & 15];
    }
    cml[0][tid] = M;
    cml[1][tid] = L;
  }
  __syncthreads();
  // 8 columns of a row of this CTA's partial, joined over its WK warps
  auto joined = [&](int r, int c8, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
#pragma unroll
    for (int k = 0; k < WK; ++k) {
      const float f = fac_s[k][r];
      if (f == 0.f) continue;            // a warp that saw nothing (or nothing that counts)
      const float* po = part + ((size_t)((r >> 4) + k * WM) * 16 + (r & 15)) * OLD + c8;
      const float4 x = reinterpret_cast<const float4*>(po)[0], y = reinterpret_cast<const float4*>(po)[1];
      v[0] += f * x.x, v[1] += f * x.y, v[2] += f * x.z, v[3] += f * x.w;
      v[4] += f * y.x, v[5] += f * y.y, v[6] += f * y.z, v[7] += f * y.w;
    }
  };
  const int live = min(RB, rows - row0);
  if (S == 1) {
    for (int i = tid; i < live * CH; i += THREADS) {
      float v[8];
      joined(i / CH, i % CH * 8, v);
      store_out(a, b, g, row0 + i / CH, i % CH * 8, HD, v, 1.f / cml[1][i / CH]);
    }
    return;
  }
  // behind the warps' partials, which other CTAs leave alone; their tiles have been read once all are here
  const Joiner jn{part + NW * 16 * OLD, ml_s, S, RB / S, OLD};
  cg::cluster_group cl = cg::this_cluster();
  cl.sync();
  for (int i = tid; i < live * CH; i += THREADS) {
    float v[8];
    const int r = i / CH, c = i % CH;
    joined(r, c * 8, v);
    float4* p = jn.row(cl, z, r) + c * 2;
    p[0] = make_float4(v[0], v[1], v[2], v[3]);
    p[1] = make_float4(v[4], v[5], v[6], v[7]);
    if (c == 0) jn.send_ml(cl, z, r, cml[0][r], cml[1][r]);
  }
  cl.sync();                             // nothing remote after this
  for (int i = tid; i < (live - z + S - 1) / S * CH; i += THREADS) {
    float v[8];
    const float L = jn.join(i / CH, i % CH * 8, v);
    store_out(a, b, g, row0 + z + i / CH * S, i % CH * 8, HD, v, 1.f / L);
  }
}

template <int WM>
int launch_tree(const TreeArgs& a, int B, cudaStream_t st) {
  static DeviceOnce attr;
  UTTT_TRY(run_once_per_device(attr, [] {
    return cuda_status(cudaFuncSetAttribute(attn_tree_kernel<WM>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            tree_smem<WM>()));
  }));
  const int blocks = (a.N * a.rep + 16 * WM - 1) / (16 * WM);
  UTTT_REQUIRE((long long)a.n_kv * blocks <= 65535, UTTT_ERR_UNSUPPORTED);
  const int S = tree_split((long long)B * a.n_kv * blocks, (a.W + TR_KT - 1) / TR_KT + 1, WM == 8 ? 1 : 2, 4, 1);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(S, a.n_kv * blocks, B);
  cfg.blockDim = dim3(tree_threads<WM>());
  cfg.dynamicSmemBytes = tree_smem<WM>();
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = S;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  at[1] = pdl_attribute();
  cfg.attrs = at;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, attn_tree_kernel<WM>, a) != cudaSuccess) return launch_status();
  return launch_status();
}

// ---------------------------------------------------------------------------
// The same on tcgen05 (head dim 64 and 128).
//
// One CTA takes 128 rows (TMEM lanes).  Tile by tile: S = Q K^T into one of two
// TMEM buffers; the thread that owns a row reads its 64 scores, keeps the running
// maximum and sum, and writes P_hi and P_lo (BF16, packed in pairs) over the same
// 64 columns, from where they enter O += P V as the A operand; O stays in TMEM.
// O is rescaled only when a row's maximum grows by more than 2^8 (weights up to
// 2^8 lose nothing: P_hi / P_lo and the FP32 sums are relative).  Warp 0 issues the
// TMA loads, warp 1 the MMAs, warps 2-5 own a row per thread; they also rotate Q
// and, in one CTA of the cluster, the drafted keys, which are its first tile.
// Two CTAs share an SM, each with 256 of its 512 TMEM columns.  A third would wait for
// columns while its cluster's other CTAs hold theirs at a barrier, and two clusters could
// wait for each other for good, so a CTA never asks for less than a third of an SM's shared
// memory (97 KB at head dim 128; 64 needs 49 KB and takes 77).
// ---------------------------------------------------------------------------
constexpr int TT_THREADS = 192;
constexpr int TT_SM_SMEM = 228 * 1024;   // shared memory of an SM, of which every CTA takes 1 KB more than it asks for
constexpr int TT_STATIC_SMEM = 4096;     // no less than the kernel's own shared variables
constexpr float TT_GROWTH = 8.f;         // log2 of the growth that a rescaling waits for

template <int HD>
struct TtLayout {
  static constexpr int BLK = HD / 64;             // 64-column blocks of a head vector
  static constexpr int Q_BYTES = 128 * HD * 2;    // per block [128 rows][128 B], K-major SW128
  static constexpr int TILE = TR_KT * HD * 2;     // per block [64 keys][128 B]
  static constexpr int K0 = Q_BYTES, V0 = Q_BYTES + 2 * TILE;   // two slots each
  static constexpr int OLD = HD + 4;              // row stride of the partial outputs (floats)
  static constexpr int USED = Q_BYTES + 4 * TILE > 128 * OLD * 4 ? Q_BYTES + 4 * TILE : 128 * OLD * 4;
  static constexpr int SMEM = 1024 + USED > TT_SM_SMEM / 3 ? 1024 + USED : TT_SM_SMEM / 3;
  static_assert(3 * (SMEM + 1024) > TT_SM_SMEM, "a third CTA must not fit an SM");
  static_assert(2 * (SMEM + 1024 + TT_STATIC_SMEM) <= TT_SM_SMEM, "two CTAs must fit an SM");
};

// D[tmem] (+)= A[tmem] * B[smem]^T (kind::f16): A is 128 lanes of packed BF16 pairs
__device__ __forceinline__ void mma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// whether the phase with this parity has completed (does not wait)
__device__ __forceinline__ bool mbar_test(uint32_t bar_addr, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar_addr), "r"(parity)
      : "memory");
  return ok != 0;
}
constexpr uint32_t kMaxLoadPolls = 1u << 26;   // of some tens of cycles: far beyond any launch
// one thread of a converged warp
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// two FP32 numbers that one instruction works on
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2_get(F2 x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v)); }
__device__ __forceinline__ F2 f2_fma(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 f2_add(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// grid (S, n_kv * row blocks, B), cluster (S, 1, 1): CTA z takes tiles [nt * z / S, nt * (z + 1) / S) of the nt
// tiles: tile 0 holds the drafted keys, tile t > 0 the ring's places 64 (t - 1) ..
template <int HD>
__global__ void __launch_bounds__(TT_THREADS, 2) attn_tree_tc_kernel(const __grid_constant__ CUtensorMap tmK,
                                                                     const __grid_constant__ CUtensorMap tmV,
                                                                     const TreeArgs a) {
  using LY = TtLayout<HD>;
  constexpr int CH = HD / 8;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t k_full[2], v_full[2], k_empty[2], v_empty[2], s_full[2], p_full[2], ready;
  __shared__ uint32_t tmem_slot;
  __shared__ u64 anc_s[2][TR_KT], bad_keys, bad_tree;
  __shared__ int jump_s[2][TR_KT], depth_s[TR_KT], deepest;
  __shared__ float ml_s[128][2];         // of the rows that the cluster sends
  __shared__ u64 bad_mask[8];            // ring tiles with non-finite values: their keys ...
  __shared__ int bad_tile[8], n_bad;     // ... and numbers
  __shared__ uint64_t drained;
  __shared__ int expired;                // whether a wait has given up: the rows become NaN then
  uint8_t* base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t *sQ = base, *sK = base + LY::K0, *sV = base + LY::V0;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int S = gridDim.x, z = blockIdx.x, b = a.b0 + blockIdx.z;
  const int g = blockIdx.y % a.n_kv, row0 = blockIdx.y / a.n_kv * 128;
  const int N = a.N, rep = a.rep, W = a.W;
  // A launch that joins the one before it starts as soon as that one's CTAs have: they waited for what came before
  // both, so all of it is complete.  Only a wait of its own would let this grid see it; instead every thread takes a
  // fence at device scope, which drops what this SM may hold of older values, for its own loads and for its tile
  // copies, before it reads anything.  The launch ends after the one before it, so that what comes next waits for both.
  if (a.joins)
    fence_device();
  else
    pdl_wait();
  const int ti = tid - 64;               // warps 2-5: 0 .. 127
  const int par_i = ti >= 0 && ti < N ? a.parents[(size_t)b * N + ti] : -1;
  const int n = a.n_nodes ? min(a.n_nodes[b], N) : N;
  const int p0 = a.pos[b], sl = a.slot[b];
  const int rows = n * rep;
  if (row0 >= rows || sl < 0 || sl >= a.n_slots || p0 < 0) {   // the same in the whole cluster
    if (a.joins) pdl_wait();
    return;
  }
  const int nvalid = min(p0, W), nt = (nvalid + TR_KT - 1) / TR_KT + 1;
  const int t_lo = (int)((long long)nt * z / S), t_hi = (int)((long long)nt * (z + 1) / S), cnt = t_hi - t_lo;
  const bool has_tree = t_lo == 0 && cnt > 0;
  const int act = 32 * ((min(128, rows - row0) + 31) / 32);   // threads that own rows; warps of padding rows rest
  // sequence i of the CTA is tile t_lo + i in slot i & 1; fills of a slot by TMA before it
  auto tma_fills = [&](int i) { return (i >> 1) - (has_tree && !(i & 1) ? 1 : 0); };

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], act);
    }
    mbar_init(&ready, 128);
    mbar_init(&drained, 1);
    fence_mbarrier_init();
    n_bad = expired = 0;
    bad_tree = 0ull;
    deepest = 0;
  }
  if (ti >= 0) prefetch_nodes<HD>(ti, 128, n, b, g, p0, a);
  if (warp == 1) tmem_alloc(&tmem_slot, 256);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // Not before this CTA has its TMEM: a matrix product that starts early takes its own and keeps it until this grid ends.
  pdl_trigger();
  const uint32_t tmem = tmem_slot, tO = tmem + 128;   // S / P: two buffers of 64 columns, O: HD columns
  int ik = 0, iv = 0;                    // key and value tiles that this thread has asked for
  bool leader = false;                   // whether it issues the MMAs

  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
      const int head = sl * a.n_kv + g;
      auto load = [&](const CUtensorMap* tm, uint8_t* ring, uint64_t* full, int i) {
        if (has_tree && i == 0) return;  // written by warps 2-5
        const int s = i & 1;
        mbar_arrive_expect_tx(&full[s], LY::TILE);
#pragma unroll
        for (int h = 0; h < LY::BLK; ++h)
          tma_load_3d(ring + s * LY::TILE + h * 8192, tm, &full[s], h * 64, (t_lo + i - 1) * TR_KT, head);
      };
      // keys and values each as soon as their own slot is free: keys' slots are released by the scores, a tile
      // period before the values'
      auto free_slot = [&](uint64_t* empty, int i) {
        return i < 2 || mbar_test(smem_u32(&empty[i & 1]), ((i >> 1) - 1) & 1);
      };
      for (uint32_t polls = 0; (ik < cnt || iv < cnt) && polls < a.max_polls; ++polls) {
        if ((polls & 1023u) == 1023u && status_set(&expired)) break;
        if (ik < cnt && free_slot(k_empty, ik)) load(&tmK, sK, k_full, ik++);
        if (iv < cnt && free_slot(v_empty, iv)) load(&tmV, sV, v_full, iv++);
      }
      if (ik < cnt || iv < cnt) set_status(&expired, UTTT_ERR_TIMEOUT);
    }
  } else if (warp == 1) {
    if (cnt > 0) {
      // The whole warp runs this loop and one elected thread issues, so that descriptors stay in uniform registers
      // (under a branch on the lane every MMA cost about 70 cycles to issue).  A descriptor's start address, in
      // units of 16 bytes, is its low bits and moves by constants.
      const uint32_t id_s = idesc_bf16(128, 64, false, false);   // A = Q K-major, B = K K-major
      const uint32_t id_o = idesc_bf16(128, HD, false, true);    // A = P in TMEM, B = V MN-major
      const uint64_t qd = sdesc_sw128(smem_u32(sQ), 16, 1024), kd = sdesc_sw128(smem_u32(sK), 16, 1024),
                     vd = sdesc_sw128(smem_u32(sV), 8192, 1024);
      const uint32_t tS = __shfl_sync(0xffffffffu, tmem, 0);
      leader = elect_one();
      mbar_wait(&ready, 0, &expired);
      __syncwarp();
      auto issue_s = [&](int i) {
        const int s = i & 1;
        if (!(has_tree && i == 0)) mbar_wait(&k_full[s], tma_fills(i) & 1, &expired);
        // P of sequence i - 2 has left this buffer
        if (i >= 2) mbar_wait(&v_empty[s], ((i >> 1) - 1) & 1, &expired);
        tc_fence_after();
        const uint64_t ks = kd + (uint64_t)(s * (LY::TILE >> 4));
        if (leader) {
#pragma unroll
          for (int k = 0; k < HD / 16; ++k)
            mma_bf16(tS + s * 64, qd + ((k >> 2) * 16384 + (k & 3) * 32) / 16,
                     ks + ((k >> 2) * 8192 + (k & 3) * 32) / 16, id_s, k > 0 ? 1u : 0u);
          mma_commit(&s_full[s]);
          mma_commit(&k_empty[s]);
        }
      };
      issue_s(0);
      for (int i = 0; i < cnt; ++i) {
        if (i + 1 < cnt) issue_s(i + 1);
        const int s = i & 1;
        if (!(has_tree && i == 0)) mbar_wait(&v_full[s], tma_fills(i) & 1, &expired);
        mbar_wait(&p_full[s], (i >> 1) & 1, &expired);
        tc_fence_after();
        const uint64_t vs = vd + (uint64_t)(s * (LY::TILE >> 4));
        const uint32_t pa = tS + s * 64;
        if (leader) {
#pragma unroll
          for (int k = 0; k < 8; ++k)    // P_hi V (columns 0 .. 31), then P_lo V (32 .. 63): 8 columns per 16 keys
            mma_bf16_ts(tS + 128, pa + k * 8, vs + (k & 3) * 2048 / 16, id_o, (i > 0 || k > 0) ? 1u : 0u);
          mma_commit(&v_empty[s]);
        }
      }
    }
  } else {
    // ---- every node's path, as in attn_tree_kernel
    if (ti < TR_KT) {
      anc_s[0][ti] = 1ull << ti;
      jump_s[0][ti] = ti < n && par_i >= 0 && par_i < ti ? par_i : -1;
    }
    named_bar(1, 128);
#pragma unroll
    for (int k = 0; k < 6; ++k) {
      if (ti < TR_KT) {
        const int j = jump_s[k & 1][ti];
        anc_s[(k & 1) ^ 1][ti] = anc_s[k & 1][ti] | (j >= 0 ? anc_s[k & 1][j] : 0ull);
        jump_s[(k & 1) ^ 1][ti] = j >= 0 ? jump_s[k & 1][j] : -1;
      }
      named_bar(1, 128);
    }
    if (ti < TR_KT) {
      u64 m = anc_s[0][ti];
      const int d = __popcll(m) - 1;
      depth_s[ti] = d;
      if (ti < n && d > 0) atomicMax(&deepest, d);
      if (d >= W)
        for (u64 rest = m; rest; rest &= rest - 1) {
          const int j = __ffsll((long long)rest) - 1;
          if (d - (__popcll(anc_s[0][j]) - 1) >= W) m &= ~(1ull << j);
        }
      anc_s[1][ti] = m;
    }
    named_bar(1, 128);
    // ---- Q, and the drafted keys and values (the rows behind the last warp of rows are never looked at)
    const __nv_bfloat16* qrows = a.qkv + (size_t)b * N * a.qkv_ld;
    const int v_col = (a.n_kv * (rep + 1) + g) * HD;
    const size_t ring0 = ((size_t)sl * a.n_kv + g) * (size_t)W * HD;
    auto put = [&](uint8_t* t, int blk, int r, int c, uint4 v) {
      *reinterpret_cast<uint4*>(t + (c >> 3) * blk + sw128_offset(r, (c & 7) * 16)) = v;
    };
    rope_nodes<HD>(
        ti, 128, n, b, g, p0, row0, act, has_tree, a, &bad_tree, [&](int node) { return depth_s[node]; },
        [&](int r, int c, uint4 v) { put(sQ, 16384, r, c, v); },
        [&](int r, int c, uint4 v) { put(sK, 8192, r, c, v); },
        [&](int r, int c, uint4 v) { put(sV, 8192, r, c, v); });
    fence_proxy_async_smem();
    mbar_arrive(&ready);

    // ---- one row per thread: row i = node i / rep, head i % rep of the group
    const int quad = warp & 3, i_row = quad * 32 + lane, row = row0 + i_row;
    const bool valid = row < rows, active = i_row < act;
    const int node = valid ? row / rep : 0, dep = depth_s[node];
    const u64 anc = anc_s[1][node];
    const int next = p0 % W, max_dep = deepest;
    const uint32_t trow = (uint32_t)(quad * 32) << 16;
    float m = -INFINITY, l = 0.f;
    for (int i = 0; active && i < cnt; ++i) {
      const int t = t_lo + i, s = i & 1, j0 = (t - 1) * TR_KT;
      const bool is_tree = t == 0;
      // keys that not every row sees: the tree's, the ring's behind the last valid place and around the window's
      // edge.  Values that must not reach the rows that do not see them leave the product (finite_values).
      const bool edge = !is_tree && (j0 + TR_KT > nvalid || (j0 <= next + max_dep && j0 + TR_KT > next) ||
                                     j0 <= next - W + max_dep);
      u64 seen = is_tree ? anc : ~0ull;
      // scores i are issued once values i - 2 have been used: after this wait v_full's phase can be told
      mbar_wait(&s_full[s], (i >> 1) & 1, &expired);
      tc_fence_after();
      // (tcgen05's loads and stores need the warp's lanes together: after every part that lanes may leave one by one)
      if (edge) {
        const u64 valid_keys = bit_range(0, nvalid - j0), some = hidden_places(j0, next, W, max_dep) & valid_keys;
        seen = valid_keys & ~hidden_places(j0, next, W, dep);
        mbar_wait(&v_full[s], tma_fills(i) & 1, &expired);
        auto at = [&](int r, int c) {
          return reinterpret_cast<uint4*>(sV + s * LY::TILE + (c >> 3) * 8192 + sw128_offset(r, (c & 7) * 16));
        };
        for (int k = (nvalid - j0) * CH + i_row; k < TR_KT * CH; k += act)   // places never written
          *at(k / CH, k % CH) = make_uint4(0, 0, 0, 0);
        if (some != 0ull) {
          if (i_row == 0) bad_keys = 0ull;
          named_bar(2, act);
          finite_values<HD>(i_row, act, some, &bad_keys, at);
          named_bar(2, act);
          if (i_row == 0 && bad_keys != 0ull && n_bad < 8) {   // at most three tiles around the edge
            bad_mask[n_bad] = bad_keys;
            bad_tile[n_bad++] = t;
          }
        }
        fence_proxy_async_smem();
      }
      __syncwarp();
      float sv[64];
#pragma unroll
      for (int c = 0; c < 64; c += 16)
        tmem_ld16(tmem + s * 64 + c + trow, *reinterpret_cast<float(*)[16]>(&sv[c]));
      tmem_wait_ld();
      if (edge || is_tree) {
#pragma unroll
        for (int c = 0; c < 64; ++c)
          if (!((c < 32 ? (uint32_t)seen : (uint32_t)(seen >> 32)) >> (c & 31) & 1u)) sv[c] = -INFINITY;
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < 64; c += 2) mx[(c >> 1) & 3] = max3(mx[(c >> 1) & 3], sv[c], sv[c + 1]);
      const float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale_log2;
      const bool grow = mt > m + TT_GROWTH || m == -INFINITY;
      if (__any_sync(0xffffffffu, grow && m != -INFINITY)) {
        // O of this warp's rows holds sequences .. i - 1: their MMAs end first
        if (i > 0) mbar_wait(&v_empty[(i - 1) & 1], ((i - 1) >> 1) & 1, &expired);
        tc_fence_after();
        __syncwarp();
        const float c = grow && m != -INFINITY ? exp2f(m - mt) : 1.f;
        l *= c;
#pragma unroll
        for (int k = 0; k < HD; k += 16) {
          float ov[16];
          uint32_t ou[16];
          tmem_ld16(tO + k + trow, ov);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e) ou[e] = __float_as_uint(ov[e] * c);
          tmem_st16(tO + k + trow, ou);
        }
      }
      if (grow) m = mt;
      const float ref = m == -INFINITY ? 0.f : m;   // nothing seen yet: every weight below is 0
      // The special-function unit computes 16 powers a cycle on an SM, 512 cycles for a tile of 128 rows.  (Powers by
      // polynomials on the FMA pipe made the tile slower: an eighth of them by 1 %, a quarter by 5 %, half by 17 %;
      // a warp of its own per scheduler is bound by what it issues.)
      F2 sum[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
      const F2 sc = f2(a.scale_log2, a.scale_log2), off = f2(-ref, -ref), minus = f2(-1.f, -1.f);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t hi[16], lo[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          F2 p = f2_fma(f2(sv[h * 32 + 2 * e], sv[h * 32 + 2 * e + 1]), sc, off);
          float x, y;
          f2_get(p, x, y);
          x = exp2f(x);
          y = exp2f(y);
          p = f2(x, y);
          sum[e & 1] = f2_add(sum[e & 1], p);
          hi[e] = pack_bf16x2(x, y);
          p = f2_fma(f2(bf16_lo(hi[e]), bf16_hi(hi[e])), minus, p);
          f2_get(p, x, y);
          lo[e] = pack_bf16x2(x, y);
        }
        tmem_st16(tmem + s * 64 + h * 16 + trow, hi);
        tmem_st16(tmem + s * 64 + 32 + h * 16 + trow, lo);
      }
      {
        float x, y;
        f2_get(f2_add(sum[0], sum[1]), x, y);
        l += x + y;
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&p_full[s]);
    }

    // ---- O -> BF16 rows of out, or partials for the cluster
    if (active && cnt > 0) mbar_wait(&v_empty[(cnt - 1) & 1], ((cnt - 1) >> 1) & 1, &expired);
    tc_fence_after();
    named_bar(1, 128);                   // bad_* is complete, no tile is in use any more
    if (status_set(&expired)) m = 0.f, l = __int_as_float(0x7fffffff);
    if (S > 1) cg::this_cluster().sync();   // every CTA has read its tiles: rows may be sent over them
    const Joiner jn{reinterpret_cast<float*>(base), ml_s, S, 128 / S, LY::OLD};
    cg::cluster_group cl = cg::this_cluster();
    if (active) {
      const float inv = 1.f / l;
      const bool any_bad = bad_tree != 0ull || n_bad > 0;
      if (S > 1 && valid) jn.send_ml(cl, z, i_row, m, l);
      float4* far = jn.row(cl, z, i_row);
      __syncwarp();
      __nv_bfloat16* dst = a.out + ((size_t)b * N + node) * a.out_ld + (size_t)(g * rep + row % rep) * HD;
#pragma unroll 1
      for (int k = 0; k < HD; k += 32) {
        float ov[32];
        if (cnt > 0) {
          tmem_ld16(tO + k + trow, *reinterpret_cast<float(*)[16]>(&ov[0]));
          tmem_ld16(tO + k + 16 + trow, *reinterpret_cast<float(*)[16]>(&ov[16]));
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) ov[e] = 0.f;
        }
        if (any_bad)
          for (int q = -1; q < n_bad; ++q) {   // the tree's, then the ring tiles'
            const int t = q < 0 ? 0 : bad_tile[q];
            u64 rest = q < 0 ? (has_tree ? bad_tree & anc : 0ull)
                             : bad_mask[q] & ~hidden_places((t - 1) * TR_KT, next, W, dep);
            for (; rest; rest &= rest - 1) {
              const int key = __ffsll((long long)rest) - 1;
              const __nv_bfloat16* v = t == 0 ? qrows + (size_t)key * a.qkv_ld + v_col
                                              : a.vring + ring0 + (size_t)((t - 1) * TR_KT + key) * HD;
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                const float x = __bfloat162float(v[k + e]);
                if ((__float_as_uint(x) & 0x7f800000u) == 0x7f800000u) ov[e] += x;
              }
            }
          }
        if (!valid) {                    // a row of padding: it only takes part in the warp's loads
        } else if (S > 1) {
#pragma unroll
          for (int e = 0; e < 32; e += 4) far[(k + e) / 4] = make_float4(ov[e], ov[e + 1], ov[e + 2], ov[e + 3]);
        } else if (a.vec_out) {
#pragma unroll
          for (int e = 0; e < 32; e += 8)
            *reinterpret_cast<uint4*>(dst + k + e) =
                make_uint4(pack_bf16x2(ov[e] * inv, ov[e + 1] * inv), pack_bf16x2(ov[e + 2] * inv, ov[e + 3] * inv),
                           pack_bf16x2(ov[e + 4] * inv, ov[e + 5] * inv), pack_bf16x2(ov[e + 6] * inv, ov[e + 7] * inv));
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) dst[k + e] = __float2bfloat16(ov[e] * inv);
        }
        __syncwarp();                    // the lanes part above; a load from tensor memory needs them together
      }
    }
  }
  __syncwarp();
  if (S > 1 && warp < 2) cg::this_cluster().sync();   // the same barrier, for the warps that issued
  tc_fence_before();
  __syncthreads();
  if (expired != 0) {                    // the same for the whole CTA
    // After a wait that expired copies and MMAs may still be under way: they end before their memory is given back.
    for (int i = max(0, ik - 2); i < ik; ++i)
      if (!(has_tree && i == 0)) mbar_wait_limit(&k_full[i & 1], tma_fills(i) & 1, nullptr, kMaxPolls);
    for (int i = max(0, iv - 2); i < iv; ++i)
      if (!(has_tree && i == 0)) mbar_wait_limit(&v_full[i & 1], tma_fills(i) & 1, nullptr, kMaxPolls);
    if (leader) {
      mma_commit(&drained);
      mbar_wait_limit(&drained, 0, nullptr, kMaxPolls);
    }
    if (tid == 0) set_status(a.status, UTTT_ERR_TIMEOUT);
    __syncthreads();
  }
  if (warp == 1) tmem_dealloc(tmem, 256);
  if (S == 1) {
    if (a.joins) pdl_wait();
    return;
  }
  cg::this_cluster().sync();             // all rows have arrived; nothing remote after this
  const Joiner jn{reinterpret_cast<float*>(base), ml_s, S, 128 / S, LY::OLD};
  const int live = min(128, rows - row0);
  for (int i = tid; i < (live - z + S - 1) / S * CH; i += TT_THREADS) {
    float v[8];
    const float L = jn.join(i / CH, i % CH * 8, v);
    store_out(a, b, g, row0 + z + i / CH * S, i % CH * 8, HD, v, 1.f / L);
  }
  if (a.joins) pdl_wait();
}

template <int HD>
int launch_tree_tc(const TreeArgs& a, int B, cudaStream_t st) {
  using LY = TtLayout<HD>;
  static DeviceOnce attr;
  UTTT_TRY(run_once_per_device(attr, [] {
    return cuda_status(
        cudaFuncSetAttribute(attn_tree_tc_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, LY::SMEM));
  }));
  // the rings as [slots * n_kv][W][hd]: places past W read as zeros
  CUtensorMap tmK, tmV;
  const uint64_t dims[3] = {(uint64_t)HD, (uint64_t)a.W, (uint64_t)a.n_slots * a.n_kv};
  const uint64_t str[2] = {(uint64_t)HD * 2, (uint64_t)a.W * HD * 2};
  const uint32_t box[3] = {64, TR_KT, 1};
  UTTT_TRY(make_tmap_bf16(&tmK, a.kring, 3, dims, str, box));
  UTTT_TRY(make_tmap_bf16(&tmV, a.vring, 3, dims, str, box));
  const int blocks = (a.N * a.rep + 127) / 128;
  UTTT_REQUIRE((long long)a.n_kv * blocks <= 65535, UTTT_ERR_UNSUPPORTED);
  auto launch = [&](int b0, int n, int S, int joins) {
    TreeArgs part = a;
    part.b0 = b0;
    part.joins = joins;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(S, a.n_kv * blocks, n);
    cfg.blockDim = dim3(TT_THREADS);
    cfg.dynamicSmemBytes = LY::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = S;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    at[1] = pdl_attribute();
    cfg.attrs = at;
    cfg.numAttrs = 2;
    if (cudaLaunchKernelEx(&cfg, attn_tree_tc_kernel<HD>, tmK, tmV, part) != cudaSuccess) return launch_status();
    return launch_status();
  };
  const int tiles = (a.W + TR_KT - 1) / TR_KT + 1, per = a.n_kv * blocks, slots = 2 * num_sms();
  const int S = tree_split((long long)B * per, tiles, 2, 4, 1);
  // A last wave with few CTAs would take as long as a full one: its rows are a launch of their own, split over
  // clusters, that fills the SMs which the full waves leave (64 rows of 16 nodes at the 1.58B heads, 320 CTAs on 296
  // places, window 512: 32.5 us in one launch, 22 us for the 59 rows of one wave).
  const int full = S == 1 ? (int)((long long)B * per / slots * slots / per) : 0, rest = B - full;
  if (full > 0 && rest > 0 && (long long)rest * per * 2 <= slots) {
    UTTT_TRY(launch(0, full, 1, 0));
    return launch(full, rest, tree_split((long long)rest * per, tiles, 2, 4, 1), 1);
  }
  return launch(0, B, S, 0);
}

// One warp per row; lane l holds nodes l and l + 32.  From node 0 on, the path goes to the lowest later child
// whose token is the pick after its parent.
__global__ void tree_accept_kernel(int B, int N, const int* __restrict__ tokens, const int* __restrict__ parents,
                                   const int* __restrict__ n_nodes, const int* __restrict__ picks,
                                   int* __restrict__ path, int* __restrict__ n_path, int* __restrict__ next) {
  const int b = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (b >= B) return;
  const int n = n_nodes ? min(max(n_nodes[b], 0), N) : N;
  int tok[2], par[2], pick[2], step[2] = {-1, -1};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int i = lane + 32 * k;
    const size_t o = (size_t)b * N + i;
    tok[k] = i < n ? tokens[o] : 0;
    par[k] = i < n ? parents[o] : -2;    // -2: no child of any node
    pick[k] = i < n ? picks[o] : 0;
  }
  int cur = 0, len = 0, want = -1;
  while (n > 0) {
    if (lane == (len & 31)) step[len >> 5] = cur;
    ++len;
    want = __shfl_sync(0xffffffffu, cur < 32 ? pick[0] : pick[1], cur & 31);
    const unsigned a = __ballot_sync(0xffffffffu, par[0] == cur && lane > cur && tok[0] == want);
    const unsigned c = __ballot_sync(0xffffffffu, par[1] == cur && lane + 32 > cur && tok[1] == want);
    if (!(a | c)) break;
    cur = a ? __ffs(a) - 1 : __ffs(c) + 31;   // later than its parent, so the walk ends
  }
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (lane + 32 * k < N) path[(size_t)b * N + lane + 32 * k] = step[k];
  if (lane == 0) {
    n_path[b] = len;
    next[b] = want;
  }
}

}  // namespace
}  // namespace uttt

using namespace uttt;

extern "C" int uttt_attn_tree_status(int B, int N, int n_heads, int n_kv, int hd, int W, int n_slots, int n_pos,
                                     const void* qkv, int qkv_ld, const int* parents, const int* n_nodes, const int* pos,
                                     const int* slot, const void* k_ring, const void* v_ring, const float* rope_cos,
                                     const float* rope_sin, void* k_tree, void* v_tree, void* out, int out_ld,
                                     int* status, unsigned max_polls, void* stream) {
  UTTT_REQUIRE(B > 0 && N > 0 && n_heads > 0 && n_kv > 0 && hd > 0 && W > 0 && n_slots > 0 && n_pos > 0,
               UTTT_ERR_INVALID);
  UTTT_REQUIRE(qkv && parents && pos && slot && k_ring && v_ring && rope_cos && rope_sin && k_tree && v_tree && out,
               UTTT_ERR_INVALID);
  UTTT_REQUIRE(n_heads % n_kv == 0 && n_heads / n_kv <= TR_MAX_REP && N <= TR_MAX_N, UTTT_ERR_UNSUPPORTED);
  UTTT_REQUIRE(hd == 32 || hd == 64 || hd == 128, UTTT_ERR_UNSUPPORTED);
  // places of a ring are told by differences of up to twice the window, in ints
  UTTT_REQUIRE(B <= 65535 && n_kv <= 65535 && W <= 1 << 30, UTTT_ERR_UNSUPPORTED);
  UTTT_REQUIRE(qkv_ld >= (n_heads + 2 * n_kv) * hd && out_ld >= n_heads * hd, UTTT_ERR_INVALID);
  cudaStream_t st = (cudaStream_t)stream;
  ProfScope ps(UTTT_PROF_ATTN, st);
  auto at16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  UTTT_REQUIRE(at16(k_ring) && at16(v_ring) && at16(k_tree) && at16(v_tree), UTTT_ERR_UNSUPPORTED);
  TreeArgs a;
  a.qkv = (const __nv_bfloat16*)qkv;
  a.parents = parents;
  a.n_nodes = n_nodes;
  a.pos = pos;
  a.slot = slot;
  a.kring = (const __nv_bfloat16*)k_ring;
  a.vring = (const __nv_bfloat16*)v_ring;
  a.cos_t = rope_cos;
  a.sin_t = rope_sin;
  a.ktree = (__nv_bfloat16*)k_tree;
  a.vtree = (__nv_bfloat16*)v_tree;
  a.out = (__nv_bfloat16*)out;
  a.qkv_ld = qkv_ld;
  a.N = N;
  a.n_kv = n_kv;
  a.rep = n_heads / n_kv;
  a.W = W;
  a.n_slots = n_slots;
  a.n_pos = n_pos;
  a.out_ld = out_ld;
  a.scale_log2 = 1.4426950408889634f / sqrtf((float)hd);
  a.vec_in = at16(qkv) && qkv_ld % 8 == 0 && at16(rope_cos) && at16(rope_sin);
  a.vec_out = at16(out) && out_ld % 8 == 0;
  a.b0 = a.joins = 0;
  a.status = status;
  a.max_polls = max_polls ? max_polls : kMaxLoadPolls;
  if (hd == 128) return launch_tree_tc<128>(a, B, st);
  if (hd == 64) return launch_tree_tc<64>(a, B, st);
  const int rows = N * a.rep;
  if (rows <= 16) return launch_tree<1>(a, B, st);
  if (rows <= 32) return launch_tree<2>(a, B, st);
  if (rows <= 64) return launch_tree<4>(a, B, st);
  return launch_tree<8>(a, B, st);
}

extern "C" int uttt_attn_tree(int B, int N, int n_heads, int n_kv, int hd, int W, int n_slots, int n_pos,
                              const void* qkv, int qkv_ld, const int* parents, const int* n_nodes, const int* pos,
                              const int* slot, const void* k_ring, const void* v_ring, const float* rope_cos,
                              const float* rope_sin, void* k_tree, void* v_tree, void* out, int out_ld,
                              void* stream) {
  return uttt_attn_tree_status(B, N, n_heads, n_kv, hd, W, n_slots, n_pos, qkv, qkv_ld, parents, n_nodes, pos, slot,
                               k_ring, v_ring, rope_cos, rope_sin, k_tree, v_tree, out, out_ld, nullptr, 0, stream);
}

extern "C" int uttt_tree_accept(int B, int N, const int* tokens, const int* parents, const int* n_nodes,
                                const int* picks, int* path, int* n_path, int* next, void* stream) {
  UTTT_REQUIRE(B > 0 && N > 0 && tokens && parents && picks && path && n_path && next, UTTT_ERR_INVALID);
  UTTT_REQUIRE(N <= TR_MAX_N, UTTT_ERR_UNSUPPORTED);
  tree_accept_kernel<<<(B + 3) / 4, 128, 0, (cudaStream_t)stream>>>(B, N, tokens, parents, n_nodes, picks, path,
                                                                    n_path, next);
  return launch_status();
}
