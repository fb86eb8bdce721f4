// Closing a KV cache behind an accepted path: slot base[b] + path[b, k] moves to slot base[b] + k, k < counts[b], for
// the keys and values of up to kKeepTensors / 2 layers in one launch.  Pure data movement, bounded by memory (large
// caches) or by the launch.
//
// path[b] ascends, so path[b, k] >= k, and a source behind the first n entries of the path lies behind the first n
// destinations.  A thread owns one vector of channels of a (row, head) and walks along the path, reading eight
// sources before it writes their destinations; no other thread touches its channels.
#include "dependent.cuh"
#include "kv_cache.cuh"

namespace tsa {

namespace {
constexpr int kKeepThreads = 128, kKeepBatch = 8;
}

template <typename V>
__global__ void __launch_bounds__(kKeepThreads) kv_keep_kernel(const __grid_constant__ KvKeep a) {
  wait_for_previous();
  let_next_start();
  const int which = blockIdx.z & 1;  // keys or values
  const int64_t vectors = a.row_bytes[which] / (int)sizeof(V);
  const int64_t item = (int64_t)blockIdx.x * kKeepThreads + threadIdx.x;
  const int b = blockIdx.y;
  const int64_t h = item / vectors, c = item % vectors;
  if (h >= a.heads) return;
  const int64_t base = a.base[b];
  const int n = min(a.nodes, a.counts[b]);
  char* row = reinterpret_cast<char*>(a.data[blockIdx.z]) + b * a.stride[which][0] + h * a.stride[which][1] +
              c * (int)sizeof(V);
  const int32_t* path = a.path + b * a.path_stride;
  for (int k0 = 0; k0 < n; k0 += kKeepBatch) {
    V v[kKeepBatch];
    bool move[kKeepBatch];
#pragma unroll
    for (int u = 0; u < kKeepBatch; ++u) {
      const int k = k0 + u;
      move[u] = false;
      if (k < n) {
        const int64_t from = path[k];
        move[u] = from > k && base >= 0 && base + from < a.capacity;
        if (move[u]) v[u] = *reinterpret_cast<const V*>(row + (base + from) * a.stride[which][2]);
      }
    }
#pragma unroll
    for (int u = 0; u < kKeepBatch; ++u)
      if (move[u]) *reinterpret_cast<V*>(row + (base + k0 + u) * a.stride[which][2]) = v[u];
  }
}

template <typename V>
static cudaError_t launch_keep(const KvKeep& a, cudaStream_t st) {
  const int64_t items = a.heads * (int64_t)(a.row_bytes[0] > a.row_bytes[1] ? a.row_bytes[0] : a.row_bytes[1]) / (int)sizeof(V);
  const dim3 grid((unsigned)((items + kKeepThreads - 1) / kKeepThreads), a.batch, a.tensors);
  return launch_dependent(kv_keep_kernel<V>, grid, dim3(kKeepThreads), 0, st, a);
}

cudaError_t kv_keep(const KvKeep& a, cudaStream_t st) {
  uint64_t bits = 0;  // the widest vector that every address, stride and row allows
  for (int i = 0; i < a.tensors; ++i) bits |= reinterpret_cast<uint64_t>(a.data[i]);
  for (int w = 0; w < 2; ++w)
    bits |= (uint64_t)a.stride[w][0] | (uint64_t)a.stride[w][1] | (uint64_t)a.stride[w][2] | (uint64_t)a.row_bytes[w];
  if (bits % 16 == 0) return launch_keep<uint4>(a, st);
  if (bits % 8 == 0) return launch_keep<uint2>(a, st);
  if (bits % 4 == 0) return launch_keep<uint32_t>(a, st);
  if (bits % 2 == 0) return launch_keep<uint16_t>(a, st);
  return launch_keep<uint8_t>(a, st);
}

// Positions of drafted nodes: the committed tokens plus the node's depth; -1 for padded nodes.
__global__ void tree_positions_kernel(const int32_t* parents, int64_t stride, const int32_t* lens, int nodes,
                                      int32_t* positions) {
  wait_for_previous();
  let_next_start();
  const int b = blockIdx.x;
  const int64_t base = lens[b];
  for (int node = threadIdx.x; node < nodes; node += blockDim.x) {
    int i = node, depth = 0;
    const int32_t* up = parents + b * stride;
    for (;;) {
      const int above = up[i];
      if (above == -1) break;
      if (above < 0 || above >= i) {
        depth = -1;
        break;
      }
      i = above;
      ++depth;
    }
    positions[(int64_t)b * nodes + node] = depth < 0 ? -1 : (int32_t)(base + depth);
  }
}

cudaError_t tree_positions(const int32_t* parents, int64_t stride, const int32_t* lens, int batch, int nodes,
                           int32_t* positions, cudaStream_t st) {
  return launch_dependent(tree_positions_kernel, dim3(batch), dim3(64), 0, st, parents, stride, lens, nodes, positions);
}

}  // namespace tsa
