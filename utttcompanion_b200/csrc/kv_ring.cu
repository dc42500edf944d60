// Copies between and into the KV rings of all layers at once: the accepted path
// of a drafted tree (uttt_kv_ring_commit) and whole rings from one persona slot
// to others (uttt_kv_ring_fork).  A ring (slots, n_kv, W, hd) holds position p at
// place p % W; the layers' rings lie layer_stride elements apart.
//
// Both are pure copies in 16-byte pieces, bound by HBM: each kept byte is read
// and written once.  16 personas' full rings of the 1.58B shape (34 layers, 713 MB)
// to other slots: 223 us, 6.40 TB/s.  A path's few nodes (at most 64 of a head) and a
// short prompt's ring are bound by the call itself, 9 us.  A piece of a head's ring
// is 1024 copies of 16 bytes, 4 per thread, so that even one short ring spreads over
// the SMs.
#include <new>

#include "common.cuh"
#include "host_util.cuh"

namespace uttt {
namespace {

// grid (layers * 2, B): tensor blockIdx.x of row blockIdx.y; V = hd / 8 pieces of 16 bytes per head vector
__global__ void ring_commit_kernel(int N, int n_kv, int V, int W, int n_slots, const uint4* __restrict__ ktree,
                                   const uint4* __restrict__ vtree, long long tree_stride, uint4* __restrict__ kring,
                                   uint4* __restrict__ vring, long long ring_stride, const int* __restrict__ pos,
                                   const int* __restrict__ slot, const int* __restrict__ path,
                                   const int* __restrict__ n_path) {
  const int b = blockIdx.y, layer = blockIdx.x >> 1;
  const int sl = slot[b], p0 = pos[b], n = min(n_path[b], N);
  if (sl < 0 || sl >= n_slots || p0 < 0) return;
  const uint4* src = ((blockIdx.x & 1) ? vtree : ktree) + (size_t)layer * tree_stride + (size_t)b * n_kv * N * V;
  uint4* dst = ((blockIdx.x & 1) ? vring : kring) + (size_t)layer * ring_stride + (size_t)sl * n_kv * W * V;
  const int first = max(0, n - W);       // of a path longer than the window the last W stay
  for (int i = threadIdx.x; i < (n - first) * n_kv * V; i += blockDim.x) {
    const int c = i % V, g = (i / V) % n_kv, t = first + i / (V * n_kv);
    const int node = path[(size_t)b * N + t];
    if (node < 0 || node >= N) continue;
    dst[((size_t)g * W + (int)(((long long)p0 + t) % W)) * V + c] = src[((size_t)g * N + node) * V + c];
  }
}

constexpr int FORK_PAIRS = 128;          // pairs per launch, passed by value
struct ForkPairs {
  int src[FORK_PAIRS], dst[FORK_PAIRS], n[FORK_PAIRS];
};

// grid (pieces of a head's ring, layers * 2 * n_kv, pairs)
__global__ void ring_fork_kernel(ForkPairs pairs, int n_kv, int V, int W, uint4* __restrict__ kring,
                                 uint4* __restrict__ vring, long long ring_stride) {
  const int pr = blockIdx.z, g = blockIdx.y % n_kv, lt = blockIdx.y / n_kv;
  uint4* base = ((lt & 1) ? vring : kring) + (size_t)(lt >> 1) * ring_stride;
  const uint4* src = base + ((size_t)pairs.src[pr] * n_kv + g) * W * V;
  uint4* dst = base + ((size_t)pairs.dst[pr] * n_kv + g) * W * V;
  const int total = pairs.n[pr] * V;
  for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < total; i += gridDim.x * blockDim.x) dst[i] = src[i];
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
}  // namespace uttt

using namespace uttt;

extern "C" int uttt_kv_ring_commit(int n_layers, int B, int N, int n_kv, int hd, int W, int n_slots,
                                   const void* k_tree, const void* v_tree, long long tree_stride, void* k_ring,
                                   void* v_ring, long long ring_stride, const int* pos, const int* slot,
                                   const int* path, const int* n_path, void* stream) {
  UTTT_REQUIRE(n_layers > 0 && B > 0 && N > 0 && n_kv > 0 && hd > 0 && W > 0 && n_slots > 0, UTTT_ERR_INVALID);
  UTTT_REQUIRE(k_tree && v_tree && k_ring && v_ring && pos && slot && path && n_path, UTTT_ERR_INVALID);
  UTTT_REQUIRE(tree_stride >= (long long)B * n_kv * N * hd && ring_stride >= (long long)n_slots * n_kv * W * hd,
               UTTT_ERR_INVALID);
  UTTT_REQUIRE(hd % 8 == 0 && tree_stride % 8 == 0 && ring_stride % 8 == 0 && aligned16(k_tree) &&
                   aligned16(v_tree) && aligned16(k_ring) && aligned16(v_ring),
               UTTT_ERR_UNSUPPORTED);
  UTTT_REQUIRE(N <= 64 && B <= 65535 && n_layers <= 1 << 20 && n_kv <= 1 << 16, UTTT_ERR_UNSUPPORTED);
  UTTT_REQUIRE((long long)N * n_kv * (hd / 8) <= 1 << 30, UTTT_ERR_UNSUPPORTED);   // pieces of a row, counted in an int
  cudaStream_t st = (cudaStream_t)stream;
  ring_commit_kernel<<<dim3(2 * n_layers, B), 256, 0, st>>>(
      N, n_kv, hd / 8, W, n_slots, (const uint4*)k_tree, (const uint4*)v_tree, tree_stride / 8,
      (uint4*)k_ring, (uint4*)v_ring, ring_stride / 8, pos, slot, path, n_path);
  return launch_status();
}

extern "C" int uttt_kv_ring_fork(int n_layers, int n_pairs, int n_kv, int hd, int W, int n_slots, void* k_ring,
                                 void* v_ring, long long ring_stride, const int* src, const int* dst,
                                 const int* end_pos, void* stream) {
  UTTT_REQUIRE(n_layers > 0 && n_pairs > 0 && n_kv > 0 && hd > 0 && W > 0 && n_slots > 0, UTTT_ERR_INVALID);
  UTTT_REQUIRE(k_ring && v_ring && src && dst && ring_stride >= (long long)n_slots * n_kv * W * hd,
               UTTT_ERR_INVALID);
  UTTT_REQUIRE(hd % 8 == 0 && ring_stride % 8 == 0 && aligned16(k_ring) && aligned16(v_ring), UTTT_ERR_UNSUPPORTED);
  // the kernel counts a head's 16-byte pieces in an int, a grid's stride past the last one
  UTTT_REQUIRE((long long)n_layers * 2 * n_kv <= 65535 && (long long)W * (hd / 8) <= 1 << 30 && n_slots <= 1 << 30,
               UTTT_ERR_UNSUPPORTED);
  // Pairs run in rounds: one goes once no other waiting pair still reads its destination, so chains (5 -> 3,
  // 7 -> 5) read what was there before the call.  Everything is checked before the first launch.
  int* buf = new (std::nothrow) int[(size_t)2 * n_slots + n_pairs];
  UTTT_REQUIRE(buf, UTTT_ERR_INVALID);
  int *reads = buf, *written = buf + n_slots, *round = written + n_slots, rounds = 0;
  for (size_t i = 0; i < (size_t)2 * n_slots; ++i) buf[i] = 0;
  int status = UTTT_OK, left = 0;
  for (int i = 0; i < n_pairs && status == UTTT_OK; ++i) {
    round[i] = -1;
    if (src[i] < 0 || src[i] >= n_slots || dst[i] < 0 || dst[i] >= n_slots || (end_pos && end_pos[i] < 0) ||
        written[dst[i]]++)
      status = UTTT_ERR_INVALID;
    else if (src[i] != dst[i]) {
      ++reads[src[i]];
      ++left;
    }
  }
  while (status == UTTT_OK && left > 0) {
    int took = 0;
    for (int i = 0; i < n_pairs; ++i)
      if (round[i] < 0 && src[i] != dst[i] && reads[dst[i]] == 0) {
        round[i] = rounds;
        ++took;
      }
    for (int i = 0; i < n_pairs; ++i)
      if (round[i] == rounds) --reads[src[i]];
    if (took == 0) status = UTTT_ERR_INVALID;   // a cycle: slots that would swap
    left -= took;
    ++rounds;
  }
  cudaStream_t st = (cudaStream_t)stream;
  const int V = hd / 8;
  for (int r = 0; r < rounds && status == UTTT_OK; ++r) {
    ForkPairs p;
    int k = 0, longest = 0;
    for (int i = 0; i <= n_pairs && status == UTTT_OK; ++i) {
      if (i < n_pairs && round[i] == r) {
        const int n = end_pos && end_pos[i] < W ? end_pos[i] : W;
        if (n > 0) {
          p.src[k] = src[i];
          p.dst[k] = dst[i];
          p.n[k++] = n;
          longest = n > longest ? n : longest;
        }
      }
      if (k == FORK_PAIRS || (i == n_pairs && k > 0)) {
        const int pieces = (longest * V + 1023) / 1024;
        ring_fork_kernel<<<dim3(pieces < 64 ? pieces : 64, n_layers * 2 * n_kv, k), 256, 0, st>>>(
            p, n_kv, V, W, (uint4*)k_ring, (uint4*)v_ring, ring_stride / 8);
        status = launch_status();
        k = longest = 0;
      }
    }
  }
  delete[] buf;
  return status;
}
