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
// Kernel.  The rep query heads of a KV head and the nodes stack into the rows of
// one matrix product (row = node * rep + head), so a ring is read once for all
// of them.  One CTA takes up to 128 rows and streams its share of the keys
// through shared memory in 64-key tiles (cp.async, three tiles in flight); the
// drafted keys are the last tile, RoPE'd in place.  WM warps stack along the rows (16
// each) and WK along the keys of a tile, so that a few rows still use every warp;
// each keeps its running maximum, sum and unnormalised output in registers.  With
// few rows in the batch a cluster of S CTAs splits the keys.  The partials meet in
// (distributed) shared memory at the end.
// The products run on mma.sync (16 x 8 x 16): at 16 to 128 rows a CTA is bound by
// the ring's bytes (a ring of 512 x 128 keys and values is 256 KB for 2 * 2 * 64 *
// 512 * 128 operations at 64 rows), a tcgen05 tile would hold mostly padding at the
// usual 16 to 64 rows and leave the softmax of a row to a single thread.
// The probabilities enter the second product as two BF16 parts, P_hi = bf16(P) and
// P_lo = bf16(P - P_hi) (about 16 significant bits, as the prefill kernel does);
// scores, statistics and sums are FP32.
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
constexpr int TR_NS = 3;                 // tiles in flight

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

// byte offset of 16-byte chunk c of row r in a tile of HD-element rows; the XOR spreads the 8 rows of an
// ldmatrix over all banks
template <int HD>
__device__ __forceinline__ uint32_t tile_off(int r, int c) {
  return (uint32_t)(r * HD * 2 + ((HD >= 64 ? c ^ (r & 7) : c ^ ((r >> 1) & 3)) << 4));
}

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
};

// 8 elements of a row of qkv
__device__ __forceinline__ uint4 load8(const __nv_bfloat16* p, int vec) {
  if (vec) return *reinterpret_cast<const uint4*>(p);
  const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
  return make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16, h[4] | (uint32_t)h[5] << 16,
                    h[6] | (uint32_t)h[7] << 16);
}
__device__ __forceinline__ void load8f(float (&f)[8], const float* p, int vec) {
  if (vec) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = p[i];
  }
}

// rotate-half RoPE of elements i0 .. i0 + 7 (`lo`) and their partners i0 + hd / 2 .. (`hi`) of a head vector,
// rounded to BF16 as apply_rope (model/uttt_layer.py:946-958)
__device__ __forceinline__ void rope8(uint4& lo, uint4& hi, const float* cosr, const float* sinr, int i0, int half,
                                      int vec) {
  uint32_t* l = reinterpret_cast<uint32_t*>(&lo);
  uint32_t* h = reinterpret_cast<uint32_t*>(&hi);
  float cl[8], ch[8], sl[8], sh[8];
  load8f(cl, cosr + i0, vec);
  load8f(ch, cosr + i0 + half, vec);
  load8f(sl, sinr + i0, vec);
  load8f(sh, sinr + i0 + half, vec);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float yl[2], yh[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float xl = e ? bf16_hi(l[k]) : bf16_lo(l[k]), xh = e ? bf16_hi(h[k]) : bf16_lo(h[k]);
      yl[e] = bfr(xl * bfr(cl[2 * k + e])) + bfr(-xh * bfr(sl[2 * k + e]));
      yh[e] = bfr(xh * bfr(ch[2 * k + e])) + bfr(xl * bfr(sh[2 * k + e]));
    }
    l[k] = pack_bf16x2(yl[0], yl[1]);
    h[k] = pack_bf16x2(yh[0], yh[1]);
  }
}

template <int HD, int WM>
__host__ __device__ constexpr int tree_threads() { return 32 * (WM < 4 ? 4 : WM); }
template <int HD>
constexpr int tree_smem() { return TR_NS * 2 * TR_KT * HD * 2; }

// grid (S, n_kv * row blocks, B), cluster (S, 1, 1): CTA z takes tiles [nt * z / S, nt * (z + 1) / S) of the nt
// 64-key tiles (the ring's, then the tree's).
template <int HD, int WM>
__global__ void __launch_bounds__(tree_threads<HD, WM>()) attn_tree_kernel(const TreeArgs a) {
  constexpr int THREADS = tree_threads<HD, WM>(), NW = THREADS / 32, WK = NW / WM;
  constexpr int RB = 16 * WM;            // rows of the CTA
  constexpr int KW = TR_KT / WK;         // keys of a tile per warp
  constexpr int SUB = KW < 32 ? KW : 32;  // keys between two updates of the running maximum
  constexpr int CH = HD / 8, TILE = TR_KT * HD * 2;
  constexpr int OLD = HD + 4;            // row stride of the partial outputs (floats): rows shift by 4 banks
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ u64 anc_s[2][TR_KT], bad_keys;
  __shared__ int jump_s[2][TR_KT], depth_s[TR_KT];
  __shared__ float m_s[NW][16], l_s[NW][16], fac_s[WK][RB], cml[2][RB];
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
  const int nvalid = min(p0, W), nring = (nvalid + TR_KT - 1) / TR_KT, nt = nring + 1;
  const int t_lo = (int)((long long)nt * z / S), t_hi = (int)((long long)nt * (z + 1) / S);
  const size_t ring0 = ((size_t)sl * a.n_kv + g) * (size_t)W * HD;
  const __nv_bfloat16* qrows = a.qkv + (size_t)b * N * a.qkv_ld;
  const int k_col = (a.n_kv * rep + g) * HD, v_col = k_col + a.n_kv * HD;
  auto table_row = [&](int node) {
    return (size_t)min((long long)p0 + depth_s[node], (long long)a.n_pos - 1) * HD;
  };
  auto load_ring = [&](int t) {
    uint8_t* ks = smem + ((t - t_lo) % TR_NS) * 2 * TILE;
    for (int i = tid; i < TR_KT * CH; i += THREADS) {
      const int r = i / CH, c = i % CH, j = t * TR_KT + r;
      const bool ok = j < nvalid;
      const size_t o = ring0 + (size_t)(ok ? j : 0) * HD + c * 8;
      cp_async_16(ks + tile_off<HD>(r, c), a.kring + o, ok);
      cp_async_16(ks + TILE + tile_off<HD>(r, c), a.vring + o, ok);
    }
  };
  // the nodes' keys (RoPE'd) and values as the last tile; one CTA per (row, KV head) also writes them out
  auto load_tree = [&]() {
    uint8_t* ks = smem + ((nt - 1 - t_lo) % TR_NS) * 2 * TILE;
    for (int i = tid; i < TR_KT * CH / 2; i += THREADS) {
      const int r = i / (CH / 2), c = i % (CH / 2);
      uint4 k0 = make_uint4(0, 0, 0, 0), k1 = k0, v0 = k0, v1 = k0;
      if (r < n) {
        const __nv_bfloat16* x = qrows + (size_t)r * a.qkv_ld;
        k0 = load8(x + k_col + c * 8, a.vec_in);
        k1 = load8(x + k_col + HD / 2 + c * 8, a.vec_in);
        v0 = load8(x + v_col + c * 8, a.vec_in);
        v1 = load8(x + v_col + HD / 2 + c * 8, a.vec_in);
        const size_t tr = table_row(r);
        rope8(k0, k1, a.cos_t + tr, a.sin_t + tr, c * 8, HD / 2, a.vec_in);
        if (row0 == 0) {
          const size_t o = (((size_t)b * a.n_kv + g) * N + r) * HD + c * 8;
          *reinterpret_cast<uint4*>(a.ktree + o) = k0;
          *reinterpret_cast<uint4*>(a.ktree + o + HD / 2) = k1;
          *reinterpret_cast<uint4*>(a.vtree + o) = v0;
          *reinterpret_cast<uint4*>(a.vtree + o + HD / 2) = v1;
        }
      }
      *reinterpret_cast<uint4*>(ks + tile_off<HD>(r, c)) = k0;
      *reinterpret_cast<uint4*>(ks + tile_off<HD>(r, c + CH / 2)) = k1;
      *reinterpret_cast<uint4*>(ks + TILE + tile_off<HD>(r, c)) = v0;
      *reinterpret_cast<uint4*>(ks + TILE + tile_off<HD>(r, c + CH / 2)) = v1;
    }
  };
#pragma unroll
  for (int i = 0; i < TR_NS - 1; ++i) {
    if (t_lo + i < t_hi && t_lo + i < nring) load_ring(t_lo + i);
    cp_async_commit();
  }

  // ---- every node's path as a bit mask, by pointer jumping (6 doublings reach 64 ancestors)
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
    if (d >= W)                          // ancestors that have left the window
      for (u64 rest = m; rest; rest &= rest - 1) {
        const int j = __ffsll((long long)rest) - 1;
        if (d - (__popcll(anc_s[0][j]) - 1) >= W) m &= ~(1ull << j);
      }
    anc_s[1][tid] = m;
  }
  __syncthreads();

  // ---- tiles of the tree that the prologue must fill, and Q: RoPE'd rows into the last stage, then registers
#pragma unroll
  for (int i = 0; i < TR_NS - 1; ++i)
    if (t_lo + i < t_hi && t_lo + i == nt - 1) load_tree();
  uint8_t* sQ = smem + (TR_NS - 1) * 2 * TILE;
  for (int i = tid; i < RB * CH / 2; i += THREADS) {
    const int r = i / (CH / 2), c = i % (CH / 2), row = row0 + r;
    uint4 q0 = make_uint4(0, 0, 0, 0), q1 = q0;
    if (row < rows) {
      const int node = row / rep, h = g * rep + row % rep;
      const __nv_bfloat16* x = qrows + (size_t)node * a.qkv_ld + (size_t)h * HD;
      q0 = load8(x + c * 8, a.vec_in);
      q1 = load8(x + HD / 2 + c * 8, a.vec_in);
      const size_t tr = table_row(node);
      rope8(q0, q1, a.cos_t + tr, a.sin_t + tr, c * 8, HD / 2, a.vec_in);
    }
    *reinterpret_cast<uint4*>(sQ + tile_off<HD>(r, c)) = q0;
    *reinterpret_cast<uint4*>(sQ + tile_off<HD>(r, c + CH / 2)) = q1;
  }
  __syncthreads();
  uint32_t qf[HD / 16][4];
#pragma unroll
  for (int k = 0; k < HD / 16; ++k)
    ldsm4(qf[k], smem_u32(sQ) + tile_off<HD>(wm * 16 + (lane & 15), 2 * k + (lane >> 4)));

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
  const int next = p0 % W;               // the oldest place: place j holds position p0 - W + (j - next mod W)
  float o[HD / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < HD / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.f;

  for (int t = t_lo; t < t_hi; ++t) {
    cp_async_wait<TR_NS - 2>();
    __syncthreads();
    if (t + TR_NS - 1 < t_hi) {
      if (t + TR_NS - 1 < nring)
        load_ring(t + TR_NS - 1);
      else
        load_tree();
    }
    cp_async_commit();
    uint8_t* ks = smem + ((t - t_lo) % TR_NS) * 2 * TILE;
    const uint32_t ka = smem_u32(ks), va = ka + TILE;
    const bool is_tree = t == nt - 1;
    // a tile whose keys not every row sees: the tree's, the ring's last, and where the window's edge lies
    // (places 0 .. 63 behind `next`, the most that a depth can hide)
    const int rel = (t * TR_KT - next + W) % W;
    const bool edge = is_tree || t * TR_KT + TR_KT > nvalid || rel < TR_KT || rel + TR_KT > W;
    u64 bad = 0ull;
    if (edge) {
      // 0 * NaN would let a key's value reach rows that do not see it: such values leave the product and are
      // added, below, to the rows that do
      if (tid == 0) bad_keys = 0ull;
      __syncthreads();
      for (int i = tid; i < TR_KT * CH; i += THREADS) {
        uint4* p = reinterpret_cast<uint4*>(ks + TILE + tile_off<HD>(i / CH, i % CH));
        uint4 v = *p;
        if (has_nonfinite(v.x) || has_nonfinite(v.y) || has_nonfinite(v.z) || has_nonfinite(v.w)) {
          *p = make_uint4(finite_only(v.x), finite_only(v.y), finite_only(v.z), finite_only(v.w));
          atomicOr(&bad_keys, 1ull << (i / CH));
        }
      }
      __syncthreads();
      bad = bad_keys;
    }
    auto sees = [&](int e, int key) -> bool {   // whether row e of this thread sees key `key` of the tile
      if (is_tree) return (anc[e] >> key) & 1ull;
      const int j = t * TR_KT + key;
      int back = j - next;               // 0 for the oldest place
      if (back < 0) back += W;
      return j < nvalid && back > dep[e];
    };
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
          ldsm4(kf, ka + tile_off<HD>(kb + i * 16 + (lane & 7) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1)));
          mma16816(s[2 * i], qf[k], kf[0], kf[1]);
          mma16816(s[2 * i + 1], qf[k], kf[2], kf[3]);
        }
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < SUB / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[i][e] *= a.scale_log2;
          if (edge && !sees(e >> 1, kb + i * 8 + (lane & 3) * 2 + (e & 1))) s[i][e] = -INFINITY;
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
          ldsm4_t(vf, va + tile_off<HD>(kb + i * 16 + (lane & 15), 2 * cc + (lane >> 4)));
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
                                       : a.vring + ring0 + (size_t)(t * TR_KT + key) * HD;
#pragma unroll
      for (int i = 0; i < HD / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = __bfloat162float(v[i * 8 + (lane & 3) * 2 + (e & 1)]);
          if ((__float_as_uint(x) & 0x7f800000u) == 0x7f800000u && sees(e >> 1, key)) o[i][e] += x;
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
  auto store = [&](int r, int c8, const float (&v)[8], float inv) {
    const int row = row0 + r, node = row / rep, h = g * rep + row % rep;
    __nv_bfloat16* dst = a.out + ((size_t)b * N + node) * a.out_ld + (size_t)h * HD + c8;
    if (a.vec_out) {
      *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16x2(v[0] * inv, v[1] * inv), pack_bf16x2(v[2] * inv, v[3] * inv),
                                                  pack_bf16x2(v[4] * inv, v[5] * inv), pack_bf16x2(v[6] * inv, v[7] * inv));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) dst[e] = __float2bfloat16(v[e] * inv);
    }
  };
  const int live = min(RB, rows - row0);
  if (S == 1) {
    for (int i = tid; i < live * CH; i += THREADS) {
      float v[8];
      joined(i / CH, i % CH * 8, v);
      store(i / CH, i % CH * 8, v, 1.f / cml[1][i / CH]);
    }
    return;
  }
  // the CTA's own join in place (its first warp's copy), then each CTA finishes every S-th row
  if (WK > 1) {
    for (int i = tid; i < live * CH; i += THREADS) {
      float v[8];
      const int r = i / CH, c8 = i % CH * 8;
      joined(r, c8, v);
      float* po = part + ((size_t)(r >> 4) * 16 + (r & 15)) * OLD + c8;   // only this thread reads or writes it
      reinterpret_cast<float4*>(po)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(po)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
  }
  cg::cluster_group cl = cg::this_cluster();
  cl.sync();
  for (int i = tid; i < (live - z + S - 1) / S * CH; i += THREADS) {
    const int r = z + i / CH * S, c8 = i % CH * 8;
    float M = -INFINITY, L = 0.f, v[8];
    for (int k = 0; k < S; ++k) M = fmaxf(M, cl.map_shared_rank(&cml[0][0], k)[r]);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    for (int k = 0; k < S; ++k) {
      const float* ml = cl.map_shared_rank(&cml[0][0], k);
      const float mk = ml[r];
      if (mk == -INFINITY) continue;     // a CTA whose keys this row does not see
      const float f = exp2f(mk - M);
      L += f * ml[RB + r];
      const float* po = cl.map_shared_rank(part, k) + ((size_t)(r >> 4) * 16 + (r & 15)) * OLD + c8;
      const float4 x = reinterpret_cast<const float4*>(po)[0], y = reinterpret_cast<const float4*>(po)[1];
      v[0] += f * x.x, v[1] += f * x.y, v[2] += f * x.z, v[3] += f * x.w;
      v[4] += f * y.x, v[5] += f * y.y, v[6] += f * y.z, v[7] += f * y.w;
    }
    store(r, c8, v, 1.f / L);
  }
  cl.sync();                             // no CTA leaves while another still reads its partial
}

template <int HD, int WM>
int launch_tree(const TreeArgs& a, int B, cudaStream_t st) {
  static DeviceOnce attr;
  UTTT_TRY(run_once_per_device(attr, [] {
    return cuda_status(cudaFuncSetAttribute(attn_tree_kernel<HD, WM>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            tree_smem<HD>()));
  }));
  const int blocks = (a.N * a.rep + 16 * WM - 1) / (16 * WM);
  UTTT_REQUIRE((long long)a.n_kv * blocks <= 65535, UTTT_ERR_UNSUPPORTED);
  // split the keys over a cluster while the batch leaves SMs idle (at least two tiles per CTA)
  const long long ctas = (long long)B * a.n_kv * blocks;
  const int tiles = (a.W + TR_KT - 1) / TR_KT + 1;
  int S = 1;
  while (S < 8 && ctas * S < 2LL * num_sms() && tiles / (2 * S) >= 2) S *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(S, a.n_kv * blocks, B);
  cfg.blockDim = dim3(tree_threads<HD, WM>());
  cfg.dynamicSmemBytes = tree_smem<HD>();
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = S;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  at[1] = pdl_attribute();
  cfg.attrs = at;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, attn_tree_kernel<HD, WM>, a) != cudaSuccess) return launch_status();
  return launch_status();
}

// ---------------------------------------------------------------------------
// The same on tcgen05, for many rows (head dim 64 or 128).
//
// One CTA takes 128 rows (TMEM lanes).  Tile by tile: S = Q K^T into one of two
// TMEM buffers; the thread that owns a row reads its 64 scores, keeps the running
// maximum and sum, and writes P_hi and P_lo (BF16, packed in pairs) over the same
// 64 columns, from where they enter O += P V as the A operand; O stays in TMEM.
// O is rescaled only when a row's maximum grows by more than 2^8 (weights up to
// 2^8 lose nothing: P_hi / P_lo and the FP32 sums are relative).  Warp 0 issues the
// TMA loads, warp 1 the MMAs, warps 2-5 own a row per thread; they also rotate Q
// and, in one CTA of the cluster, the drafted keys, which are its first tile.
// Two CTAs of 96 KB and 256 TMEM columns share an SM.
// ---------------------------------------------------------------------------
constexpr int TT_THREADS = 192;
constexpr float TT_GROWTH = 8.f;         // log2 of the growth that a rescaling waits for

template <int HD>
struct TtLayout {
  static constexpr int BLK = HD / 64;             // 64-column blocks of a head vector
  static constexpr int Q_BYTES = 128 * HD * 2;    // per block [128 rows][128 B], K-major SW128
  static constexpr int TILE = TR_KT * HD * 2;     // per block [64 keys][128 B]
  static constexpr int K0 = Q_BYTES, V0 = Q_BYTES + 2 * TILE;   // two slots each
  static constexpr int OLD = HD + 4;              // row stride of the partial outputs (floats)
  static constexpr int USED = Q_BYTES + 4 * TILE > 128 * OLD * 4 ? Q_BYTES + 4 * TILE : 128 * OLD * 4;
  static constexpr int SMEM = 1024 + USED;
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
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

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
  __shared__ u64 anc_s[2][TR_KT], bad_keys;
  __shared__ int jump_s[2][TR_KT], depth_s[TR_KT];
  __shared__ float cml[2][128];
  __shared__ u64 bad_mask[8];            // tiles with non-finite values: their keys ...
  __shared__ int bad_tile[8], n_bad;     // ... and numbers
  uint8_t* base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t *sQ = base, *sK = base + LY::K0, *sV = base + LY::V0;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int S = gridDim.x, z = blockIdx.x, b = blockIdx.z;
  const int g = blockIdx.y % a.n_kv, row0 = blockIdx.y / a.n_kv * 128;
  const int N = a.N, rep = a.rep, W = a.W;
  pdl_wait();
  pdl_trigger();
  const int n = a.n_nodes ? min(a.n_nodes[b], N) : N;
  const int p0 = a.pos[b], sl = a.slot[b];
  const int rows = n * rep;
  if (row0 >= rows || sl < 0 || sl >= a.n_slots || p0 < 0) return;   // the same in the whole cluster
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
    fence_mbarrier_init();
    n_bad = 0;
  }
  if (warp == 1) tmem_alloc(&tmem_slot, 256);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot, tO = tmem + 128;   // S / P: two buffers of 64 columns, O: HD columns

  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
      const int head = sl * a.n_kv + g;
      auto load = [&](const CUtensorMap* tm, uint8_t* ring, uint64_t* full, uint64_t* empty, int i) {
        if (i >= cnt || (has_tree && i == 0)) return;
        const int s = i & 1;
        if (i >= 2) mbar_wait(&empty[s], ((i >> 1) - 1) & 1, nullptr);
        mbar_arrive_expect_tx(&full[s], LY::TILE);
#pragma unroll
        for (int h = 0; h < LY::BLK; ++h)
          tma_load_3d(ring + s * LY::TILE + h * 8192, tm, &full[s], h * 64, (t_lo + i - 1) * TR_KT, head);
      };
      load(&tmK, sK, k_full, k_empty, 0);
      for (int i = 0; i < cnt; ++i) {
        load(&tmK, sK, k_full, k_empty, i + 1);
        load(&tmV, sV, v_full, v_empty, i);
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && cnt > 0) {
      const uint32_t id_s = idesc_bf16(128, 64, false, false);   // A = Q K-major, B = K K-major
      const uint32_t id_o = idesc_bf16(128, HD, false, true);    // A = P in TMEM, B = V MN-major
      const uint32_t qa = smem_u32(sQ);
      mbar_wait(&ready, 0, nullptr);
      auto issue_s = [&](int i) {
        const int s = i & 1;
        if (!(has_tree && i == 0)) mbar_wait(&k_full[s], tma_fills(i) & 1, nullptr);
        // P of sequence i - 2 has left this buffer
        if (i >= 2) mbar_wait(&v_empty[s], ((i >> 1) - 1) & 1, nullptr);
        tc_fence_after();
        const uint32_t ka = smem_u32(sK + s * LY::TILE);
#pragma unroll
        for (int k = 0; k < HD / 16; ++k)
          mma_bf16(tmem + s * 64, sdesc_sw128(qa + (k >> 2) * 16384 + (k & 3) * 32, 16, 1024),
                   sdesc_sw128(ka + (k >> 2) * 8192 + (k & 3) * 32, 16, 1024), id_s, k > 0 ? 1u : 0u);
        mma_commit(&s_full[s]);
        mma_commit(&k_empty[s]);
      };
      issue_s(0);
      for (int i = 0; i < cnt; ++i) {
        if (i + 1 < cnt) issue_s(i + 1);
        const int s = i & 1;
        if (!(has_tree && i == 0)) mbar_wait(&v_full[s], tma_fills(i) & 1, nullptr);
        mbar_wait(&p_full[s], (i >> 1) & 1, nullptr);
        tc_fence_after();
        const uint32_t va = smem_u32(sV + s * LY::TILE), pa = tmem + s * 64;
#pragma unroll
        for (int k = 0; k < 8; ++k)      // P_hi V (columns 0 .. 31), then P_lo V (32 .. 63): 8 columns per 16 keys
          mma_bf16_ts(tO, pa + k * 8, sdesc_sw128(va + (k & 3) * 2048, 8192, 1024), id_o,
                      (i > 0 || k > 0) ? 1u : 0u);
        mma_commit(&v_empty[s]);
      }
    }
  } else {
    const int ti = tid - 64;             // 0 .. 127
    // ---- every node's path, as in attn_tree_kernel
    const int par_i = ti < N ? a.parents[(size_t)b * N + ti] : -1;
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
      if (d >= W)
        for (u64 rest = m; rest; rest &= rest - 1) {
          const int j = __ffsll((long long)rest) - 1;
          if (d - (__popcll(anc_s[0][j]) - 1) >= W) m &= ~(1ull << j);
        }
      anc_s[1][ti] = m;
    }
    named_bar(1, 128);
    // ---- Q, and the drafted keys and values
    const __nv_bfloat16* qrows = a.qkv + (size_t)b * N * a.qkv_ld;
    const int k_col = (a.n_kv * rep + g) * HD, v_col = k_col + a.n_kv * HD;
    const size_t ring0 = ((size_t)sl * a.n_kv + g) * (size_t)W * HD;
    auto table_row = [&](int node) {
      return (size_t)min((long long)p0 + depth_s[node], (long long)a.n_pos - 1) * HD;
    };
    auto put = [&](uint8_t* t, int blk, int r, int c, uint4 v) {
      *reinterpret_cast<uint4*>(t + (c >> 3) * blk + sw128_offset(r, (c & 7) * 16)) = v;
    };
    for (int i = ti; i < 128 * CH / 2; i += 128) {
      const int r = i / (CH / 2), c = i % (CH / 2), row = row0 + r;
      uint4 q0 = make_uint4(0, 0, 0, 0), q1 = q0;
      if (row < rows) {
        const int node = row / rep;
        const __nv_bfloat16* x = qrows + (size_t)node * a.qkv_ld + (size_t)(g * rep + row % rep) * HD;
        q0 = load8(x + c * 8, a.vec_in);
        q1 = load8(x + HD / 2 + c * 8, a.vec_in);
        const size_t tr = table_row(node);
        rope8(q0, q1, a.cos_t + tr, a.sin_t + tr, c * 8, HD / 2, a.vec_in);
      }
      put(sQ, 16384, r, c, q0);
      put(sQ, 16384, r, c + CH / 2, q1);
    }
    if (has_tree) {
      for (int i = ti; i < TR_KT * CH / 2; i += 128) {
        const int r = i / (CH / 2), c = i % (CH / 2);
        uint4 k0 = make_uint4(0, 0, 0, 0), k1 = k0, v0 = k0, v1 = k0;
        if (r < n) {
          const __nv_bfloat16* x = qrows + (size_t)r * a.qkv_ld;
          k0 = load8(x + k_col + c * 8, a.vec_in);
          k1 = load8(x + k_col + HD / 2 + c * 8, a.vec_in);
          v0 = load8(x + v_col + c * 8, a.vec_in);
          v1 = load8(x + v_col + HD / 2 + c * 8, a.vec_in);
          const size_t tr = table_row(r);
          rope8(k0, k1, a.cos_t + tr, a.sin_t + tr, c * 8, HD / 2, a.vec_in);
          if (row0 == 0) {
            const size_t o = (((size_t)b * a.n_kv + g) * N + r) * HD + c * 8;
            *reinterpret_cast<uint4*>(a.ktree + o) = k0;
            *reinterpret_cast<uint4*>(a.ktree + o + HD / 2) = k1;
            *reinterpret_cast<uint4*>(a.vtree + o) = v0;
            *reinterpret_cast<uint4*>(a.vtree + o + HD / 2) = v1;
          }
        }
        put(sK, 8192, r, c, k0);
        put(sK, 8192, r, c + CH / 2, k1);
        put(sV, 8192, r, c, v0);
        put(sV, 8192, r, c + CH / 2, v1);
      }
    }
    fence_proxy_async_smem();
    mbar_arrive(&ready);

    // ---- one row per thread: row i = node i / rep, head i % rep of the group
    const int quad = warp & 3, i_row = quad * 32 + lane, row = row0 + i_row;
    const bool valid = row < rows, active = i_row < act;
    const int node = valid ? row / rep : 0, dep = depth_s[node];
    const u64 anc = anc_s[1][node];
    const int next = p0 % W;
    const uint32_t trow = (uint32_t)(quad * 32) << 16;
    float m = -INFINITY, l = 0.f;
    for (int i = 0; active && i < cnt; ++i) {
      const int t = t_lo + i, s = i & 1, j0 = (t - 1) * TR_KT;
      const bool is_tree = t == 0;
      const int rel = is_tree ? 0 : (j0 - next + W) % W;
      const bool edge = is_tree || j0 + TR_KT > nvalid || rel < TR_KT || rel + TR_KT > W;
      // scores i are issued once values i - 2 have been used: after this wait v_full's phase can be told
      mbar_wait(&s_full[s], (i >> 1) & 1, nullptr);
      tc_fence_after();
      if (edge) {
        // 0 * NaN would let a key's value reach rows that do not see it: such values leave the product and
        // are added at the end to the rows that do
        if (!is_tree) mbar_wait(&v_full[s], tma_fills(i) & 1, nullptr);
        if (i_row == 0) bad_keys = 0ull;
        named_bar(2, act);
        for (int k = i_row; k < TR_KT * CH; k += act) {
          const int r = k / CH, c = k % CH;
          uint4* p = reinterpret_cast<uint4*>(sV + s * LY::TILE + (c >> 3) * 8192 + sw128_offset(r, (c & 7) * 16));
          const uint4 v = *p;
          if (has_nonfinite(v.x) || has_nonfinite(v.y) || has_nonfinite(v.z) || has_nonfinite(v.w)) {
            *p = make_uint4(finite_only(v.x), finite_only(v.y), finite_only(v.z), finite_only(v.w));
            atomicOr(&bad_keys, 1ull << r);
          }
        }
        fence_proxy_async_smem();
        named_bar(2, act);
        if (i_row == 0 && bad_keys != 0ull && n_bad < 8) {   // at most a tree, a last tile and three of the edge
          bad_mask[n_bad] = bad_keys;
          bad_tile[n_bad++] = t;
        }
      }
      float sv[64];
#pragma unroll
      for (int c = 0; c < 64; c += 16)
        tmem_ld16(tmem + s * 64 + c + trow, *reinterpret_cast<float(*)[16]>(&sv[c]));
      tmem_wait_ld();
      float mt = -INFINITY;
      if (edge) {
#pragma unroll
        for (int c = 0; c < 64; ++c) {
          bool see;
          if (is_tree) {
            see = (anc >> c) & 1ull;
          } else {
            int back = j0 + c - next;
            if (back < 0) back += W;
            see = j0 + c < nvalid && back > dep;
          }
          if (!see) sv[c] = -INFINITY;
        }
      }
#pragma unroll
      for (int c = 0; c < 64; ++c) mt = fmaxf(mt, sv[c]);
      mt *= a.scale_log2;
      const bool grow = mt > m + TT_GROWTH || m == -INFINITY;
      if (__any_sync(0xffffffffu, grow && m != -INFINITY)) {
        // O of this warp's rows holds sequences .. i - 1: their MMAs end first
        if (i > 0) mbar_wait(&v_empty[(i - 1) & 1], ((i - 1) >> 1) & 1, nullptr);
        tc_fence_after();
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
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t hi[16], lo[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float x = exp2f(fmaf(sv[h * 32 + 2 * e], a.scale_log2, -ref));
          const float y = exp2f(fmaf(sv[h * 32 + 2 * e + 1], a.scale_log2, -ref));
          l += x + y;
          hi[e] = pack_bf16x2(x, y);
          lo[e] = pack_bf16x2(x - bf16_lo(hi[e]), y - bf16_hi(hi[e]));
        }
        tmem_st16(tmem + s * 64 + h * 16 + trow, hi);
        tmem_st16(tmem + s * 64 + 32 + h * 16 + trow, lo);
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&p_full[s]);
    }

    // ---- O -> BF16 rows of out, or partials for the cluster
    if (active && cnt > 0) mbar_wait(&v_empty[(cnt - 1) & 1], ((cnt - 1) >> 1) & 1, nullptr);
    tc_fence_after();
    named_bar(1, 128);                   // bad_* is complete, no tile is in use any more
    const float inv = 1.f / l;
    float* part = reinterpret_cast<float*>(base) + (size_t)i_row * LY::OLD;
    __nv_bfloat16* dst = a.out + ((size_t)b * N + node) * a.out_ld + (size_t)(g * rep + row % rep) * HD;
    if (active) {
#pragma unroll
      for (int k = 0; k < HD; k += 16) {
        float ov[16];
        if (cnt > 0) {
          tmem_ld16(tO + k + trow, ov);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) ov[e] = 0.f;
        }
        for (int q = 0; q < n_bad; ++q)
          for (u64 rest = bad_mask[q]; rest; rest &= rest - 1) {
            const int key = __ffsll((long long)rest) - 1, t = bad_tile[q];
            int back = (t - 1) * TR_KT + key - next;
            if (back < 0) back += W;
            const bool see = t == 0 ? (anc >> key) & 1ull : (t - 1) * TR_KT + key < nvalid && back > dep;
            if (!see) continue;
            const __nv_bfloat16* v = t == 0 ? qrows + (size_t)key * a.qkv_ld + v_col
                                            : a.vring + ring0 + (size_t)((t - 1) * TR_KT + key) * HD;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float x = __bfloat162float(v[k + e]);
              if ((__float_as_uint(x) & 0x7f800000u) == 0x7f800000u) ov[e] += x;
            }
          }
        if (S > 1) {
#pragma unroll
          for (int e = 0; e < 16; e += 4)
            *reinterpret_cast<float4*>(part + k + e) = make_float4(ov[e], ov[e + 1], ov[e + 2], ov[e + 3]);
        } else if (valid) {
          if (a.vec_out) {
#pragma unroll
            for (int e = 0; e < 16; e += 8)
              *reinterpret_cast<uint4*>(dst + k + e) =
                  make_uint4(pack_bf16x2(ov[e] * inv, ov[e + 1] * inv), pack_bf16x2(ov[e + 2] * inv, ov[e + 3] * inv),
                             pack_bf16x2(ov[e + 4] * inv, ov[e + 5] * inv),
                             pack_bf16x2(ov[e + 6] * inv, ov[e + 7] * inv));
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) dst[k + e] = __float2bfloat16(ov[e] * inv);
          }
        }
      }
    }
    cml[0][i_row] = m;
    cml[1][i_row] = l;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 256);
  if (S == 1) return;
  // every CTA finishes every S-th row of the block
  cg::cluster_group cl = cg::this_cluster();
  cl.sync();
  const int live = min(128, rows - row0);
  float* part0 = reinterpret_cast<float*>(base);
  for (int i = tid; i < (live - z + S - 1) / S * CH; i += TT_THREADS) {
    const int r = z + i / CH * S, c8 = i % CH * 8, row = row0 + r;
    float M = -INFINITY, L = 0.f, v[8];
    for (int k = 0; k < S; ++k) M = fmaxf(M, cl.map_shared_rank(&cml[0][0], k)[r]);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    for (int k = 0; k < S; ++k) {
      const float* ml = cl.map_shared_rank(&cml[0][0], k);
      const float mk = ml[r];
      if (mk == -INFINITY) continue;     // a CTA whose keys this row does not see
      const float f = exp2f(mk - M);
      L += f * ml[128 + r];
      const float* po = cl.map_shared_rank(part0, k) + (size_t)r * LY::OLD + c8;
      const float4 x = reinterpret_cast<const float4*>(po)[0], y = reinterpret_cast<const float4*>(po)[1];
      v[0] += f * x.x, v[1] += f * x.y, v[2] += f * x.z, v[3] += f * x.w;
      v[4] += f * y.x, v[5] += f * y.y, v[6] += f * y.z, v[7] += f * y.w;
    }
    const float inv = 1.f / L;
    __nv_bfloat16* dst = a.out + ((size_t)b * N + row / rep) * a.out_ld + (size_t)(g * rep + row % rep) * HD + c8;
    if (a.vec_out) {
      *reinterpret_cast<uint4*>(dst) =
          make_uint4(pack_bf16x2(v[0] * inv, v[1] * inv), pack_bf16x2(v[2] * inv, v[3] * inv),
                     pack_bf16x2(v[4] * inv, v[5] * inv), pack_bf16x2(v[6] * inv, v[7] * inv));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) dst[e] = __float2bfloat16(v[e] * inv);
    }
  }
  cl.sync();                             // no CTA leaves while another still reads its partial
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
  const long long ctas = (long long)B * a.n_kv * blocks;
  const int tiles = (a.W + TR_KT - 1) / TR_KT + 1;
  int S = 1;
  while (S < 8 && ctas * S < 2LL * num_sms() && tiles / (2 * S) >= 2) S *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(S, a.n_kv * blocks, B);
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
  if (cudaLaunchKernelEx(&cfg, attn_tree_tc_kernel<HD>, tmK, tmV, a) != cudaSuccess) return launch_status();
  return launch_status();
}

template <int HD>
int launch_tree_rows(const TreeArgs& a, int B, cudaStream_t st) {
  const int rows = a.N * a.rep;
  if constexpr (HD >= 64)
    if (rows > 32) return launch_tree_tc<HD>(a, B, st);
  if (rows <= 16) return launch_tree<HD, 1>(a, B, st);
  if (rows <= 32) return launch_tree<HD, 2>(a, B, st);
  if (rows <= 64) return launch_tree<HD, 4>(a, B, st);
  return launch_tree<HD, 8>(a, B, st);
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

extern "C" int uttt_attn_tree(int B, int N, int n_heads, int n_kv, int hd, int W, int n_slots, int n_pos,
                              const void* qkv, int qkv_ld, const int* parents, const int* n_nodes, const int* pos,
                              const int* slot, const void* k_ring, const void* v_ring, const float* rope_cos,
                              const float* rope_sin, void* k_tree, void* v_tree, void* out, int out_ld,
                              void* stream) {
  UTTT_REQUIRE(B > 0 && N > 0 && n_heads > 0 && n_kv > 0 && hd > 0 && W > 0 && n_slots > 0 && n_pos > 0,
               UTTT_ERR_INVALID);
  UTTT_REQUIRE(qkv && parents && pos && slot && k_ring && v_ring && rope_cos && rope_sin && k_tree && v_tree && out,
               UTTT_ERR_INVALID);
  UTTT_REQUIRE(n_heads % n_kv == 0 && n_heads / n_kv <= TR_MAX_REP && N <= TR_MAX_N, UTTT_ERR_UNSUPPORTED);
  UTTT_REQUIRE(hd == 32 || hd == 64 || hd == 128, UTTT_ERR_UNSUPPORTED);
  UTTT_REQUIRE(B <= 65535 && n_kv <= 65535, UTTT_ERR_UNSUPPORTED);
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
  if (hd == 32) return launch_tree_rows<32>(a, B, st);
  if (hd == 64) return launch_tree_rows<64>(a, B, st);
  return launch_tree_rows<128>(a, B, st);
}

extern "C" int uttt_tree_accept(int B, int N, const int* tokens, const int* parents, const int* n_nodes,
                                const int* picks, int* path, int* n_path, int* next, void* stream) {
  UTTT_REQUIRE(B > 0 && N > 0 && tokens && parents && picks && path && n_path && next, UTTT_ERR_INVALID);
  UTTT_REQUIRE(N <= TR_MAX_N, UTTT_ERR_UNSUPPORTED);
  tree_accept_kernel<<<(B + 3) / 4, 128, 0, (cudaStream_t)stream>>>(B, N, tokens, parents, n_nodes, picks, path,
                                                                    n_path, next);
  return launch_status();
}
