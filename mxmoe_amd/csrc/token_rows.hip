// Tokens sorted by expert and back, and the gradients of both; the gradient of the routing.
//
//   permute            rows[row(t, s)] = hidden[t]                       row(t, s): stable order by (expert, t * topk + s), ids out of range last
//   permute, backward  grad_hidden[t] = sum_s grad_rows[row(t, s)]       (the kernel of the way back, without weights)
//   unpermute          out[t] = sum_s w[t, s] rows[row(t, s)] + shared[t]
//   unpermute, backward  grad_rows[row(t, s)] = w[t, s] grad_out[t],  grad_w[t, s] = <grad_out[t], rows[row(t, s)]>
//   routing, backward  from the weights' gradient to the logits'
//
// The reference sorts with torch::sort + index_select (mxmoe/kernels/src/ref_bind.cu:47-64), leaves the way back an empty stub (:66) and has no gradients.
//
// All of them are bound by memory.  The kernels run over TOKENS, not over sorted rows: a token's own row (hidden, out, grad_out) is read or written once
// for all of its slots, every sorted row once, and every sum stays inside one thread or workgroup: no atomics on memory, results do not depend on the order
// of anything.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <string>

#include "../../include/mxmoe_amd.h"
#include "include/mxmoe_launch.hpp"
#include "include/mxmoe_perm.hpp"
#include "include/mxmoe_rows.hpp"
#include "include/mxmoe_vec8.hpp"

namespace mxmoe {

// ---- permute ----
//
// Two questions: where a slot's row goes, and the copy.  A workgroup takes `per_wg` tokens, finds the rows of their slots and copies each token to them, so that the
// copy needs no launch of its own.  A slot's row = (rows of smaller experts) + (slots of its expert before the workgroup's first) + (its rank among the workgroup's).
// The counts come from
//   direct   the ids themselves, all of them read by every workgroup (up to kDirectSlots: 16 KB of 4-byte ids; one launch);
//   counted  a first launch that counts the experts in chunks of kCountChunk slots: the workgroup sums the table's rows and counts the slots of its own chunk that
//            lie before its first (two launches, up to kCountedMax table entries: 32 KB from L2 a workgroup);
//   scanned  the same with a launch between that turns the table's rows into prefixes (three launches, beside which the copy of that many rows is long).
constexpr int kDirectSlots = 4096;
constexpr int kCountChunk = 1024;
constexpr int kCountedMax = 8192;
constexpr int kWgSlots = 256;  // slots of a workgroup's tokens, at most

struct PermuteArgs {
  const uint8_t* hidden;
  long ld;                 // bytes from one token's row to the next
  const void* ids;
  int T, topk, E, nbits;
  unsigned row_bytes;
  int per_wg;              // tokens a workgroup
  int keep_tail;           // leave the rows of dropped slots as they are (else they are cleared)
  uint8_t* rows;
  int32_t* row_of_slot;
  int64_t* recv;
  int64_t* perm;           // token of every sorted row, or null
  const int32_t* table;    // [E + 1][stride]: slots of every expert (E: of none) in every chunk; scanned: those before the chunk
  const int32_t* totals;   // scanned: [E + 1]
  int chunks, stride;
};

template <typename ID>
__device__ __forceinline__ int bucket_of(const void* ids, int i, int E) {
  const ID e = reinterpret_cast<const ID*>(ids)[i];
  return e >= 0 && e < (ID)E ? (int)e : E;  // (compared in its own width: a 64-bit id past 2^32 names no expert either)
}

template <typename ID>
__global__ void __launch_bounds__(256) permute_count_kernel(const void* ids, int total, int E, int32_t* table, int stride) {
  extern __shared__ int32_t cnt[];
  for (int e = threadIdx.x; e <= E; e += 256) cnt[e] = 0;
  __syncthreads();
  const int base = blockIdx.x * kCountChunk;
#pragma unroll
  for (int i = 0; i < kCountChunk; i += 256) {
    const int idx = base + i + threadIdx.x;
    if (idx < total) atomicAdd(&cnt[bucket_of<ID>(ids, idx, E)], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e <= E; e += 256) table[(long)e * stride + blockIdx.x] = cnt[e];
}

// one wave per bucket: its row of the table becomes the exclusive prefix over the chunks
__global__ void __launch_bounds__(64) permute_scan_kernel(int32_t* table, int chunks, int stride, int32_t* totals) {
  int32_t* row = table + (long)blockIdx.x * stride;
  int carry = 0;
  for (int c0 = 0; c0 < chunks; c0 += 64) {
    const int c = c0 + threadIdx.x;
    const int v = c < chunks ? row[c] : 0;
    const int inc = wave_inclusive_scan(v);
    if (c < chunks) row[c] = carry + inc - v;
    carry += wave_last(inc);
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

typedef uint32_t v4u __attribute__((ext_vector_type(4)));
struct __attribute__((packed, aligned(2))) Bytes16 {  // 16 bytes of a row, which starts at any element
  v4u v;
};

enum PermuteCounts { kDirect, kCounted, kScanned };

template <typename ID, int COUNTS>
__global__ void __launch_bounds__(256) permute_kernel(const PermuteArgs a) {
  extern __shared__ int32_t lds[];
  const int E = a.E, nb = E + 1, tid = threadIdx.x, lane = tid & 63;
  int32_t* run = lds;              // [E + 1] next row of every bucket among this workgroup's slots
  int32_t* tot = lds + nb;         // [E + 1]
  int32_t* pos = lds + 2 * nb;     // [kWgSlots]
  const int t0 = blockIdx.x * a.per_wg, nt = min(a.per_wg, a.T - t0);
  const int i0 = t0 * a.topk, n_slots = nt * a.topk, total = a.T * a.topk;
  // the first pieces of the tokens' rows are on their way while the rows' places are found
  constexpr int U = 4;
  const unsigned P = a.row_bytes >> 4, n_pieces = nt * P;
  const uint8_t* src = a.hidden + t0 * a.ld;
  Bytes16 first[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const unsigned n = tid + 256u * u;
    if (n < n_pieces) first[u] = *reinterpret_cast<const Bytes16*>(src + n / P * a.ld + n % P * 16);
  }
  for (int e = tid; e < nb; e += 256) {
    run[e] = COUNTS == kScanned ? a.table[(long)e * a.stride + i0 / kCountChunk] : 0;
    tot[e] = COUNTS == kScanned ? a.totals[e] : 0;
  }
  __syncthreads();
  if constexpr (COUNTS == kDirect) {
    for (int i = tid; i < total; i += 256) {
      const int e = bucket_of<ID>(a.ids, i, E);
      atomicAdd(&tot[e], 1);
      if (i < i0) atomicAdd(&run[e], 1);
    }
  } else {
    if constexpr (COUNTS == kCounted) {
      const int quads = a.stride >> 2, chunk = i0 / kCountChunk;
      for (int q = tid; q < nb * quads; q += 256) {
        const int e = q / quads, b = 4 * (q % quads);
        const v4u h = *reinterpret_cast<const v4u*>(a.table + (long)e * a.stride + b);
        int all = 0, before = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // (the padding behind the last chunk holds anything)
          all += b + i < a.chunks ? (int)h[i] : 0;
          before += b + i < chunk ? (int)h[i] : 0;
        }
        if (all) atomicAdd(&tot[e], all);
        if (before) atomicAdd(&run[e], before);
      }
    }
    for (int i = i0 / kCountChunk * kCountChunk + tid; i < i0; i += 256) atomicAdd(&run[bucket_of<ID>(a.ids, i, E)], 1);
  }
  __syncthreads();
  if (tid < 64) {
    int carry = 0;
    for (int e0 = 0; e0 < nb; e0 += 64) {
      const int e = e0 + lane;
      const int v = e < nb ? tot[e] : 0;
      const int inc = wave_inclusive_scan(v);
      if (e < nb) run[e] += carry + inc - v;
      carry += wave_last(inc);
    }
  }
  if (blockIdx.x == 0)
    for (int e = tid; e < E; e += 256) a.recv[e] = tot[e];
  __syncthreads();
  for (int i = 0; i < n_slots; i += 64) {  // 64 slots at a time, in order: the order inside an expert is that of the slots
    const bool mine = tid < 64 && i + lane < n_slots;
    const int e = mine ? bucket_of<ID>(a.ids, i0 + i + lane, E) : nb;
    int p = 0, before = 0;
    uint64_t same = 0;
    if (tid < 64) {
      same = match_same(e, a.nbits);
      before = __popcll(same & ((1ull << lane) - 1));
      if (mine) p = run[e] + before;
    }
    __syncthreads();
    if (mine) {
      if (before == 0) run[e] += __popcll(same);
      pos[i + lane] = e < E ? p : -2 - p;
      a.row_of_slot[i0 + i + lane] = e < E ? p : -2 - p;
      if (a.perm && e < E) a.perm[p] = (i0 + i + lane) / a.topk;
    }
    __syncthreads();
  }
  const int k = a.topk;
  auto put = [&](unsigned token, unsigned offset, auto bytes) {
    for (int s = 0; s < k; ++s) {
      const int p = pos[token * k + s];
      if (p >= 0) *reinterpret_cast<decltype(bytes)*>(a.rows + (size_t)p * a.row_bytes + offset) = bytes;
      else if (!a.keep_tail) *reinterpret_cast<decltype(bytes)*>(a.rows + (size_t)(-2 - p) * a.row_bytes + offset) = decltype(bytes){};
    }
  };
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const unsigned n = tid + 256u * u;
    if (n < n_pieces) put(n / P, n % P * 16, first[u]);
  }
  for (unsigned n0 = 256u * U + tid; n0 < n_pieces; n0 += 256u * U) {
    Bytes16 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned n = n0 + 256u * u;
      if (n < n_pieces) v[u] = *reinterpret_cast<const Bytes16*>(src + n / P * a.ld + n % P * 16);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned n = n0 + 256u * u;
      if (n < n_pieces) put(n / P, n % P * 16, v[u]);
    }
  }
  // what a row has past its last whole 16 bytes
  const unsigned rest = (a.row_bytes & 15) >> 1;
  for (unsigned n = tid; n < nt * rest; n += 256) {
    const unsigned offset = 16 * P + 2 * (n % rest);
    put(n / rest, offset, *reinterpret_cast<const uint16_t*>(src + n / rest * a.ld + offset));
  }
}

// ---- unpermute, and permute's backward ----
//
// `tpt` threads a token (whole waves, so that a token's rows and weights are scalars), 16 bytes of every row at a time, up to eight slots' loads in flight.
// Products and sums are rounded one by one in slot order, as combine_kernel's: the same bits for fp16.
struct GatherArgs {
  const void* rows;
  long ld;
  int num_rows;
  const int32_t* row_of_slot;
  const float* weights;   // [T][topk], or null: 1
  const void* shared;     // [T] rows of K, or null
  long ld_shared;
  int T, topk, K, tpt;
  void* out;
};
template <typename T>
__global__ void __launch_bounds__(256) unpermute_kernel(const GatherArgs a) {
  constexpr int kSlots = 8;
  const int team = __builtin_amdgcn_readfirstlane((int)threadIdx.x / a.tpt);
  const int t = blockIdx.x * (256 / a.tpt) + team;
  if (t >= a.T) return;  // (no barrier below)
  const int C = (a.K + 7) >> 3;
  for (int c = threadIdx.x % a.tpt; c < C; c += a.tpt) {
    f8 acc = 0.0f;
    typename Piece<T>::raw sh{};
    if (a.shared) sh = load_piece(reinterpret_cast<const T*>(a.shared) + t * a.ld_shared, c, a.K);
    for (int s0 = 0; s0 < a.topk; s0 += kSlots) {
      int r[kSlots];
      typename Piece<T>::raw v[kSlots];
#pragma unroll
      for (int i = 0; i < kSlots; ++i) r[i] = s0 + i < a.topk ? const_load(a.row_of_slot + (long)t * a.topk + s0 + i) : -1;
#pragma unroll
      for (int i = 0; i < kSlots; ++i)
        if (r[i] >= 0 && r[i] < a.num_rows) v[i] = load_piece(reinterpret_cast<const T*>(a.rows) + r[i] * a.ld, c, a.K);
#pragma unroll
      for (int i = 0; i < kSlots; ++i)
        if (r[i] >= 0 && r[i] < a.num_rows) {
          const f8 x = Piece<T>::widen(v[i]);
          acc = acc + (a.weights ? const_load(a.weights + (long)t * a.topk + s0 + i) * x : x);
        }
    }
    if (a.shared) acc = acc + Piece<T>::widen(sh);
    store_piece(reinterpret_cast<T*>(a.out) + (long)t * a.K, c, a.K, Piece<T>::narrow(acc));
  }
}

// ---- unpermute, backward ----
//
// One workgroup of NT threads a token; S slots at a time (of a top-k of 2, 4 or more).  grad_out's piece stays in registers while it is multiplied with each slot's row (the
// weight's gradient) and by each weight (the row's gradient): one pass over everything.
struct UngatherArgs {
  const void* grad_out;
  long ld_grad;
  const void* rows;       // read only for grad_weights
  long ld;
  int num_rows;
  const int32_t* row_of_slot;
  const float* weights;
  int topk, K, keep_tail;
  void* grad_rows;
  float* grad_weights;    // or null
};
template <typename T, int NT, int S>
__global__ void __launch_bounds__(NT) unpermute_backward_kernel(const UngatherArgs a) {
  __shared__ float sums[2][S * (NT / 64)];
  const int t = blockIdx.x, C = (a.K + 7) >> 3;
  const T* g_row = reinterpret_cast<const T*>(a.grad_out) + t * a.ld_grad;
  for (int s0 = 0, turn = 0; s0 < a.topk; s0 += S, turn ^= 1) {
    int r[S];
    float w[S], dot[S];
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const long at = (long)t * a.topk + s0 + i;
      r[i] = s0 + i < a.topk ? const_load(a.row_of_slot + at) : -1;
      w[i] = s0 + i < a.topk && a.weights ? const_load(a.weights + at) : 1.0f;
      dot[i] = 0.0f;
    }
    for (int c = threadIdx.x; c < C; c += NT) {
      const auto g_raw = load_piece(g_row, c, a.K);
      typename Piece<T>::raw v[S];
      if (a.grad_weights) {
#pragma unroll
        for (int i = 0; i < S; ++i)
          if (r[i] >= 0 && r[i] < a.num_rows) v[i] = load_piece(reinterpret_cast<const T*>(a.rows) + r[i] * a.ld, c, a.K);
      }
      const f8 g = Piece<T>::widen(g_raw);
#pragma unroll
      for (int i = 0; i < S; ++i) {
        if (r[i] >= 0 && r[i] < a.num_rows) {
          if (a.grad_weights) {
            const f8 x = Piece<T>::widen(v[i]);
#pragma unroll
            for (int e = 0; e < 8; ++e) dot[i] = __builtin_fmaf(g[e], x[e], dot[i]);
          }
          store_piece(reinterpret_cast<T*>(a.grad_rows) + (long)r[i] * a.K, c, a.K, Piece<T>::narrow(w[i] * g));
        } else if (r[i] <= -2 && -2 - r[i] < a.num_rows && !a.keep_tail) {
          store_piece(reinterpret_cast<T*>(a.grad_rows) + (long)(-2 - r[i]) * a.K, c, a.K, typename Piece<T>::raw{});
        }
      }
    }
    if (!a.grad_weights) continue;
    group_sum<NT, S>(dot, sums[turn]);
#pragma unroll
    for (int i = 0; i < S; ++i)
      if ((int)threadIdx.x == i && s0 + i < a.topk) a.grad_weights[(long)t * a.topk + s0 + i] = dot[i];
  }
}

// ---- routing, backward ----
//
// p = softmax(logits) over all experts, or with `renorm` over the chosen ones (there p / sum of the chosen p); w = the chosen p.
//   inner = sum_s dw[s] p[id(s)]
//   grad_logit[j] = p[j] ( sum_{s: id(s) = j} dw[s]  -  inner ),  with renorm p[j] sum_{s: id(s) = j} (dw[s] - inner).
// G lanes a token, a power of two of at least min(E, 64) and topk, so that a lane holds a slot; experts go in rounds of G.
struct RouteGradArgs {
  const float* grad_weights;
  const void* logits;
  int dtype;
  const int32_t* ids;
  int T, E, topk, renorm, G;
  void* grad_logits;
};
__global__ void __launch_bounds__(256) route_backward_kernel(const RouteGradArgs a) {
  const int G = a.G, g = threadIdx.x & (G - 1);
  const int t = blockIdx.x * (256 / G) + (int)threadIdx.x / G;
  const bool live = t < a.T;  // (lanes without a token go along: the sums run over whole waves)
  const long base = (long)t * a.E;
  auto over_team = [&](float v, auto op) {
    for (int o = G >> 1; o > 0; o >>= 1) v = op(v, __shfl_xor(v, o, G));
    return v;
  };
  auto larger = [](float x, float y) { return fmaxf(x, y); };
  auto plus = [](float x, float y) { return x + y; };
  int id = -1;
  float dw = 0.0f, mine = -INFINITY;
  if (live && g < a.topk) {
    id = a.ids[(long)t * a.topk + g];
    if (id >= 0 && id < a.E) {
      dw = a.grad_weights[(long)t * a.topk + g];
      mine = load_of(a.dtype, a.logits, base + id);
    } else {
      id = -1;
    }
  }
  float mx = -INFINITY, sum = 0.0f;
  if (a.renorm) {
    mx = over_team(mine, larger);
    sum = over_team(id >= 0 ? expf(mine - mx) : 0.0f, plus);
  } else {
    for (int e = g; e < a.E; e += G)
      if (live) mx = fmaxf(mx, load_of(a.dtype, a.logits, base + e));
    mx = over_team(mx, larger);
    for (int e = g; e < a.E; e += G)
      if (live) sum += expf(load_of(a.dtype, a.logits, base + e) - mx);
    sum = over_team(sum, plus);
  }
  const float inner = over_team(id >= 0 ? dw * (expf(mine - mx) / sum) : 0.0f, plus);
  for (int e0 = 0; e0 < a.E; e0 += G) {
    const int e = e0 + g;
    float d = a.renorm ? 0.0f : -inner;
    bool chosen = false;
    for (int s = 0; s < a.topk; ++s) {  // (an expert that a token names twice gets both slots' gradients)
      const int of = __shfl(id, s, G);
      const float v = __shfl(dw, s, G);
      if (of == e) {
        d += a.renorm ? v - inner : v;
        chosen = true;
      }
    }
    if (live && e < a.E) {
      float grad = 0.0f;
      if (!a.renorm || chosen) grad = expf(load_of(a.dtype, a.logits, base + e) - mx) / sum * d;
      store_of(a.dtype, a.grad_logits, base + e, grad);
    }
  }
}

static int refuse(int code, const char* what) {
  last_error() = what;
  return code;
}
static int launched() {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return 0;
  last_error() = std::string("kernel launch failed: ") + hipGetErrorString(e);
  return 4;
}
static int permute_stride(long slots) { return ((int)((slots + kCountChunk - 1) / kCountChunk) + 3) & ~3; }

template <typename ID>
static int run_permute(PermuteArgs& a, int32_t* table, hipStream_t s) {
  const int total = a.T * a.topk, nb = a.E + 1;
  const size_t lds = (size_t)(2 * nb + kWgSlots) * sizeof(int32_t);
  const int grid = std::max(1, (a.T + a.per_wg - 1) / a.per_wg);  // (no tokens: the counts are still written)
  if (total <= kDirectSlots) {
    hipLaunchKernelGGL((permute_kernel<ID, kDirect>), dim3(grid), dim3(256), lds, s, a);
    return launched();
  }
  a.stride = permute_stride(total);
  a.chunks = (total + kCountChunk - 1) / kCountChunk;
  a.table = table;
  a.totals = table + (long)nb * a.stride;
  hipLaunchKernelGGL(permute_count_kernel<ID>, dim3(a.chunks), dim3(256), nb * sizeof(int32_t), s, a.ids, total, a.E, table, a.stride);
  if ((long)nb * a.stride <= kCountedMax) {
    hipLaunchKernelGGL((permute_kernel<ID, kCounted>), dim3(grid), dim3(256), lds, s, a);
  } else {
    hipLaunchKernelGGL(permute_scan_kernel, dim3(nb), dim3(64), 0, s, table, a.chunks, a.stride, table + (long)nb * a.stride);
    hipLaunchKernelGGL((permute_kernel<ID, kScanned>), dim3(grid), dim3(256), lds, s, a);
  }
  return launched();
}

template <typename T, int NT>
static void run_unpermute_backward(const UngatherArgs& a, int num_tokens, hipStream_t s) {
  if (a.topk <= 2) hipLaunchKernelGGL((unpermute_backward_kernel<T, NT, 2>), dim3(num_tokens), dim3(NT), 0, s, a);
  else if (a.topk <= 4) hipLaunchKernelGGL((unpermute_backward_kernel<T, NT, 4>), dim3(num_tokens), dim3(NT), 0, s, a);
  else hipLaunchKernelGGL((unpermute_backward_kernel<T, NT, 8>), dim3(num_tokens), dim3(NT), 0, s, a);
}

static const char* kTokenSizes = "tokens sorted by expert: tokens >= 0, 1 <= topk <= 64, 1 <= experts <= 4096, K >= 1 and at most 2^30 (token, slot) pairs";
static bool token_sizes_ok(int num_tokens, int topk, int num_experts, int K) {
  return num_tokens >= 0 && topk >= 1 && topk <= 64 && (long)num_tokens * topk <= (1l << 30) && num_experts >= 1 && num_experts <= 4096 && K >= 1 && K <= (1 << 28);
}

}  // namespace mxmoe

using namespace mxmoe;

extern "C" {

size_t mxmoe_permute_tokens_workspace_bytes(int num_tokens, int topk, int num_experts) {
  const long slots = (long)num_tokens * topk;
  if (slots <= kDirectSlots || num_experts < 1) return 0;
  return (size_t)(num_experts + 1) * (permute_stride(slots) + 1) * sizeof(int32_t);
}

int mxmoe_permute_tokens(const void* hidden, int64_t ld, int dtype, const void* topk_ids, int ids_bytes, int num_tokens, int topk, int num_experts, int K, void* rows, int keep_tail,
                         int32_t* row_of_slot, int64_t* recv_tokens_per_exp, int64_t* perm_indices, void* workspace, void* stream) {
  if (!token_sizes_ok(num_tokens, topk, num_experts, K)) return refuse(3, kTokenSizes);
  if (dtype < 0 || dtype > 2 || (ids_bytes != 4 && ids_bytes != 8) || ld < 0) return refuse(3, "rows as fp16 (0), fp32 (1) or bf16 (2), ids of 4 or 8 bytes, row strides >= 0");
  if (!recv_tokens_per_exp || (num_tokens && (!hidden || !topk_ids || !rows || !row_of_slot))) return refuse(5, "null pointer");
  if (!workspace && mxmoe_permute_tokens_workspace_bytes(num_tokens, topk, num_experts)) return refuse(5, "null pointer");
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return refuse(3, "the workspace must be 16-byte aligned");
  PermuteArgs a{};
  a.hidden = reinterpret_cast<const uint8_t*>(hidden);
  a.ld = (long)ld * (long)float_bytes(dtype);
  a.ids = topk_ids;
  a.T = num_tokens;
  a.topk = topk;
  a.E = num_experts;
  a.nbits = 1;
  while ((1 << a.nbits) <= num_experts + 1) ++a.nbits;  // buckets 0 .. E, and E + 1: lanes without a slot
  a.row_bytes = (unsigned)(K * float_bytes(dtype));
  // Tokens a workgroup: one while there are few, else 16 KB of rows, so that a table of counts is summed for several tokens at once
  const int by_rows = (int)std::max(1u, 16384u / a.row_bytes), by_tokens = std::max(1, num_tokens / 1024);
  a.per_wg = std::min({by_rows, by_tokens, kWgSlots / topk});
  a.keep_tail = keep_tail != 0;
  a.rows = reinterpret_cast<uint8_t*>(rows);
  a.row_of_slot = row_of_slot;
  a.recv = recv_tokens_per_exp;
  a.perm = perm_indices;
  int32_t* table = reinterpret_cast<int32_t*>(workspace);
  return ids_bytes == 4 ? run_permute<int32_t>(a, table, (hipStream_t)stream) : run_permute<int64_t>(a, table, (hipStream_t)stream);
}

int mxmoe_unpermute_tokens(const void* rows, int64_t ld, int num_rows, const int32_t* row_of_slot, const float* topk_weights, const void* shared, int64_t ld_shared, int dtype,
                           int num_tokens, int topk, int K, void* out, void* stream) {
  if (!token_sizes_ok(num_tokens, topk, 1, K) || num_rows < 0) return refuse(3, kTokenSizes);
  if (dtype < 0 || dtype > 2 || ld < 0 || ld_shared < 0) return refuse(3, "rows as fp16 (0), fp32 (1) or bf16 (2), row strides >= 0");
  if (num_tokens == 0) return 0;
  if ((num_rows && !rows) || !row_of_slot || !out) return refuse(5, "null pointer");
  GatherArgs a{rows, (long)ld, num_rows, row_of_slot, topk_weights, shared, (long)ld_shared, num_tokens, topk, K, 0, out};
  const int C = (K + 7) / 8;
  a.tpt = C <= 64 ? 64 : (C <= 128 ? 128 : 256);
  const dim3 grid((num_tokens + 256 / a.tpt - 1) / (256 / a.tpt));
  hipStream_t s = (hipStream_t)stream;
  if (dtype == kF16) hipLaunchKernelGGL(unpermute_kernel<_Float16>, grid, dim3(256), 0, s, a);
  else if (dtype == kF32) hipLaunchKernelGGL(unpermute_kernel<float>, grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL(unpermute_kernel<__bf16>, grid, dim3(256), 0, s, a);
  return launched();
}

int mxmoe_unpermute_tokens_backward(const void* grad_out, int64_t ld_grad, const void* rows, int64_t ld, int num_rows, const int32_t* row_of_slot, const float* topk_weights, int dtype,
                                    int num_tokens, int topk, int K, void* grad_rows, int keep_tail, float* grad_weights, void* stream) {
  if (!token_sizes_ok(num_tokens, topk, 1, K) || num_rows < 0) return refuse(3, kTokenSizes);
  if (dtype < 0 || dtype > 2 || ld < 0 || ld_grad < 0) return refuse(3, "rows as fp16 (0), fp32 (1) or bf16 (2), row strides >= 0");
  if (num_tokens == 0) return 0;
  if (!grad_out || !row_of_slot || (num_rows && !grad_rows) || (grad_weights && num_rows && !rows)) return refuse(5, "null pointer");
  const UngatherArgs a{grad_out, (long)ld_grad, rows, (long)ld, num_rows, row_of_slot, topk_weights, topk, K, keep_tail != 0, grad_rows, grad_weights};
  hipStream_t s = (hipStream_t)stream;
  const bool narrow = K <= 1024;
  if (dtype == kF16) narrow ? run_unpermute_backward<_Float16, 64>(a, num_tokens, s) : run_unpermute_backward<_Float16, 256>(a, num_tokens, s);
  else if (dtype == kF32) narrow ? run_unpermute_backward<float, 64>(a, num_tokens, s) : run_unpermute_backward<float, 256>(a, num_tokens, s);
  else narrow ? run_unpermute_backward<__bf16, 64>(a, num_tokens, s) : run_unpermute_backward<__bf16, 256>(a, num_tokens, s);
  return launched();
}

int mxmoe_route_topk_backward(const float* grad_weights, const void* router_logits, int logits_dtype, const int32_t* topk_ids, int num_tokens, int num_experts, int topk, int renormalise,
                              void* grad_logits, void* stream) {
  if (num_tokens < 0 || num_experts <= 0 || num_experts > 4096 || topk <= 0 || topk > num_experts || topk > 64 || logits_dtype < 0 || logits_dtype > 2)
    return refuse(3, "routing takes 1..4096 experts, top-k of at most min(experts, 64), logits as fp16 (0), fp32 (1) or bf16 (2)");
  if (num_tokens == 0) return 0;
  if (!grad_weights || !router_logits || !topk_ids || !grad_logits) return refuse(5, "null pointer");
  RouteGradArgs a{grad_weights, router_logits, logits_dtype, topk_ids, num_tokens, num_experts, topk, renormalise != 0, 4, grad_logits};
  while (a.G < 64 && (a.G < num_experts || a.G < topk)) a.G *= 2;
  const int per_wg = 256 / a.G;
  hipLaunchKernelGGL(route_backward_kernel, dim3((num_tokens + per_wg - 1) / per_wg), dim3(256), 0, (hipStream_t)stream, a);
  return launched();
}

}  // extern "C"
