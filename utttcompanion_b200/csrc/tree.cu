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
#include "common.cuh"
#include "host_util.cuh"

namespace uttt {
namespace {

constexpr int TR_MAX_N = 64;
constexpr int TR_MAX_REP = 8;

__device__ __forceinline__ float bfr(float x) { return __bfloat162float(__float2bfloat16(x)); }

// rotate-half RoPE of element i of a head vector x, rounded to BF16 as apply_rope (model/uttt_layer.py:946-958)
__device__ __forceinline__ float rope_elem(const __nv_bfloat16* x, int i, int hd, const float* cosr,
                                           const float* sinr) {
  const int half = hd >> 1;
  const float xi = __bfloat162float(x[i]);
  const float rot = i < half ? -__bfloat162float(x[i + half]) : __bfloat162float(x[i - half]);
  return bfr(bfr(xi * bfr(cosr[i])) + bfr(rot * bfr(sinr[i])));
}

// a parent that is not an earlier node makes a root
__device__ __forceinline__ int parent_of(const int* parents, int i) {
  const int p = parents[i];
  return p >= 0 && p < i ? p : -1;
}

// One CTA per (node, KV head, row), one warp per query head: the warp walks the visible keys with the running
// maximum and sum of the softmax, HD / 32 elements per lane.
template <int HD>
__global__ void attn_tree_kernel(const __nv_bfloat16* __restrict__ qkv, int qkv_ld, int N, int n_kv, int rep, int W,
                                 int n_slots, int n_pos, const int* __restrict__ parents,
                                 const int* __restrict__ n_nodes, const int* __restrict__ pos,
                                 const int* __restrict__ slot, const __nv_bfloat16* __restrict__ kring,
                                 const __nv_bfloat16* __restrict__ vring, const float* __restrict__ cos_t,
                                 const float* __restrict__ sin_t, float scale, __nv_bfloat16* __restrict__ ktree,
                                 __nv_bfloat16* __restrict__ vtree, __nv_bfloat16* __restrict__ out, int out_ld) {
  constexpr int E = HD / 32;
  const int node = blockIdx.x, g = blockIdx.y, b = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = n_nodes ? min(n_nodes[b], N) : N;
  const int p0 = pos[b], sl = slot[b];
  if (node >= n || sl < 0 || sl >= n_slots || p0 < 0) return;
  const int* par = parents + (size_t)b * N;
  int depth = 0;
  for (int a = parent_of(par, node); a >= 0; a = parent_of(par, a)) ++depth;
  const int n_heads = n_kv * rep, h = g * rep + warp, p = p0 + depth;
  const __nv_bfloat16* rows = qkv + (size_t)b * N * qkv_ld;
  const __nv_bfloat16* row = rows + (size_t)node * qkv_ld;
  auto table = [&](const float* t, int at) { return t + (size_t)min(at, n_pos - 1) * HD; };
  float q[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = rope_elem(row + (size_t)h * HD, lane * E + e, HD, table(cos_t, p), table(sin_t, p));
    acc[e] = 0.f;
  }
  if (warp == 0) {
    const size_t o = (((size_t)b * n_kv + g) * N + node) * HD;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = lane * E + e;
      ktree[o + i] = __float2bfloat16(
          rope_elem(row + (size_t)(n_heads + g) * HD, i, HD, table(cos_t, p), table(sin_t, p)));
      vtree[o + i] = row[(size_t)(n_heads + n_kv + g) * HD + i];
    }
  }
  auto take = [&](const float (&k)[E], const __nv_bfloat16* v) {
    float d = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) d += q[e] * k[e];
    d = warp_sum(d) * scale;
    const float mn = fmaxf(m, d), c = __expf(m - mn), pe = __expf(d - mn);
    l = l * c + pe;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = acc[e] * c + pe * __bfloat162float(v[lane * E + e]);
    m = mn;
  };
  const __nv_bfloat16* kr = kring + ((size_t)sl * n_kv + g) * (size_t)W * HD;
  const __nv_bfloat16* vr = vring + ((size_t)sl * n_kv + g) * (size_t)W * HD;
  for (int at = max(0, p - W + 1); at < p0; ++at) {
    const size_t o = (size_t)(at % W) * HD;
    float k[E];
#pragma unroll
    for (int e = 0; e < E; ++e) k[e] = __bfloat162float(kr[o + lane * E + e]);
    take(k, vr + o);
  }
  int d = depth;
  for (int a = node; a >= 0 && depth - d < W; a = parent_of(par, a), --d) {
    const __nv_bfloat16* ar = rows + (size_t)a * qkv_ld;
    float k[E];
#pragma unroll
    for (int e = 0; e < E; ++e)
      k[e] = rope_elem(ar + (size_t)(n_heads + g) * HD, lane * E + e, HD, table(cos_t, p0 + d), table(sin_t, p0 + d));
    take(k, ar + (size_t)(n_heads + n_kv + g) * HD);
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
    out[((size_t)b * N + node) * out_ld + (size_t)h * HD + lane * E + e] = __float2bfloat16(acc[e] / l);
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
  const float scale = 1.f / sqrtf((float)hd);
  const int rep = n_heads / n_kv;
  const dim3 grid(N, n_kv, B);
#define UTTT_TREE(HDV)                                                                                              \
  attn_tree_kernel<HDV><<<grid, 32 * rep, 0, st>>>(                                                                 \
      (const __nv_bfloat16*)qkv, qkv_ld, N, n_kv, rep, W, n_slots, n_pos, parents, n_nodes, pos, slot,              \
      (const __nv_bfloat16*)k_ring, (const __nv_bfloat16*)v_ring, rope_cos, rope_sin, scale, (__nv_bfloat16*)k_tree, \
      (__nv_bfloat16*)v_tree, (__nv_bfloat16*)out, out_ld)
  if (hd == 32)
    UTTT_TREE(32);
  else if (hd == 64)
    UTTT_TREE(64);
  else
    UTTT_TREE(128);
#undef UTTT_TREE
  return launch_status();
}

extern "C" int uttt_tree_accept(int B, int N, const int* tokens, const int* parents, const int* n_nodes,
                                const int* picks, int* path, int* n_path, int* next, void* stream) {
  UTTT_REQUIRE(B > 0 && N > 0 && tokens && parents && picks && path && n_path && next, UTTT_ERR_INVALID);
  UTTT_REQUIRE(N <= TR_MAX_N, UTTT_ERR_UNSUPPORTED);
  tree_accept_kernel<<<(B + 3) / 4, 128, 0, (cudaStream_t)stream>>>(B, N, tokens, parents, n_nodes, picks, path,
                                                                    n_path, next);
  return launch_status();
}
