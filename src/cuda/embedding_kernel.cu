// Embedding: out[t] = round(scale * weight[token[t]]), and the gradient of the
// table: out[v] (+)= round(scale * sum of grad[t] over the tokens t that name v).
//
// The gradient sorts the tokens' positions by row (a stable radix sort, so that
// the positions of a row stay in their order), cuts the sorted list into ranges
// and gives every block a range and a slice of the columns.  Its warps add the
// rows of a run of equal tokens in fp32 registers; a run inside a warp's part is
// written at once, one over its edges is joined in shared memory, one over the
// range's edges in the workspace by the block that arrives last.  Every sum is
// added in the tokens' order: the result does not depend on that of execution.
//
// All of it is bound by memory: a row is read once, a row of the table written
// once (and read once where it is added to).  On a B200 (6.56 TB/s for a plain
// copy), as calls among others, floors in brackets:
//   lookup, 16384 rows of 2048 fp32 into bf16              22.5 us  (17.6)
//   16384 rows of 4096 bf16 into an fp32 table of 50021    75 us    (50), 11 of them the sort, 57 the sums
//   8192 rows of 2048 bf16 into a new table of 100003      73.5 us  (67.5), the sort hidden behind the clearing
//   131072 rows of 1024 fp32 into an fp32 table of 32000   149 us   (121), 22 of them the sort, 127 the sums
//   33 rows of 770 bf16 into an fp32 table                 6.2 us, the launch and a chain of four memory latencies
#include <cooperative_groups.h>

#include <algorithm>

#include "grad_ops.h"
#include "ibcomm/communicator.h"
#include "kernels.h"
#include "vec_ops.cuh"

namespace ibcomm {
namespace dev {

// kN values at `p` (aligned to their size, 16 bytes at most) as fp32, and back.
template <typename T, int kN>
__device__ __forceinline__ void LoadValues(const T* p, float* a) {
  constexpr int kBytes = kN * static_cast<int>(sizeof(T));
  if constexpr (kBytes >= 16) {
#pragma unroll
    for (int v = 0; v < kBytes / 16; ++v) VecIO<T>::Load(Ld16(p + v * VecIO<T>::kN), a + v * VecIO<T>::kN);
  } else {
    static_assert(kBytes == 8 && sizeof(T) == 2, "half a vector of 16-bit values");
    const uint2 q = *reinterpret_cast<const uint2*>(p);
    float b[8];
    VecIO<T>::Load(make_uint4(q.x, q.y, 0, 0), b);
#pragma unroll
    for (int e = 0; e < kN; ++e) a[e] = b[e];
  }
}
template <typename T, int kN>
__device__ __forceinline__ void StoreValues(T* p, const float* a) {
  constexpr int kBytes = kN * static_cast<int>(sizeof(T));
  if constexpr (kBytes >= 16) {
#pragma unroll
    for (int v = 0; v < kBytes / 16; ++v) St16(p + v * VecIO<T>::kN, VecIO<T>::Store(a + v * VecIO<T>::kN));
  } else {
    static_assert(kBytes == 8 && sizeof(T) == 2, "half a vector of 16-bit values");
    *reinterpret_cast<uint2*>(p) = make_uint2(VecIO<T>::P2(a[0], a[1]), VecIO<T>::P2(a[2], a[3]));
  }
}

// ------------------------------------------------------------------ lookup
constexpr int kLookupThreads = 256;
constexpr int kLookupUnroll = 4;
constexpr int kLookupColumns = 512;  // of a warp, where rows do not come in vectors

template <typename TI, typename TO>
struct LookupQuantum {
  // 16 bytes of the narrower type at most: 16-bit values in eights, fp32 to fp32 in fours.
  static constexpr int kN = sizeof(TI) == 4 && sizeof(TO) == 4 ? 4 : 8;
};

template <bool kTokens64>
__device__ __forceinline__ int64_t Token(const void* tokens, uint64_t t) {
  if constexpr (kTokens64) return static_cast<const long long*>(tokens)[t];
  else return static_cast<const int*>(tokens)[t];
}

// A warp takes kLookupUnroll * 32 quanta (kN values each) of a row, all loads
// before the first store; where a row has fewer than 32, 1 << lanes of the warp's
// lanes take a row each.  The parts of a row are neighbours in the grid.  Against
// a thread per quantum, which divides to find its row: 26.7 -> 22.5 us for 16384
// rows of 2048 fp32 into bf16; two or eight quanta per lane are the same.
template <typename TI, typename TO, bool kTokens64>
__global__ void __launch_bounds__(kLookupThreads) EmbeddingKernel(const void* __restrict__ tokens, const TI* __restrict__ weight, TO* __restrict__ out,
                                                                  uint64_t num_tokens, uint32_t per_row, uint32_t parts, int lanes, uint64_t rows, uint64_t width,
                                                                  float scale) {
  constexpr int kN = LookupQuantum<TI, TO>::kN;
  const uint32_t lane = threadIdx.x & 31, group = 1u << lanes;
  const uint32_t block = blockIdx.x / parts, part = blockIdx.x - block * parts;
  const uint64_t warp = static_cast<uint64_t>(block) * (kLookupThreads / 32) + threadIdx.x / 32;
  const uint64_t t = (warp << (5 - lanes)) + (lane >> lanes);
  if (t >= num_tokens) return;
  const uint32_t first = (part * kLookupUnroll << lanes) + (lane & (group - 1));
  const int64_t id = Token<kTokens64>(tokens, t);
  const bool inside = id >= 0 && static_cast<uint64_t>(id) < rows;
  const TI* from = weight + (inside ? static_cast<uint64_t>(id) : 0) * width;
  TO* to = out + t * width;
  float a[kLookupUnroll][kN];
#pragma unroll
  for (int u = 0; u < kLookupUnroll; ++u) {
    const uint32_t q = first + (u << lanes);
#pragma unroll
    for (int e = 0; e < kN; ++e) a[u][e] = 0.f;
    if (inside && q < per_row) LoadValues<TI, kN>(from + static_cast<uint64_t>(q) * kN, a[u]);
  }
#pragma unroll
  for (int u = 0; u < kLookupUnroll; ++u) {
    const uint32_t q = first + (u << lanes);
    if (q < per_row) {
      if (inside) {  // a row that is not there is zero whatever the scale is
#pragma unroll
        for (int e = 0; e < kN; ++e) a[u][e] *= scale;
      }
      StoreValues<TO, kN>(to + static_cast<uint64_t>(q) * kN, a[u]);
    }
  }
}

// Rows that do not come in vectors, because of their width or of where they
// start: a warp copies the 16-byte words of memory that hold its columns into
// shared memory (no allocation ends inside one) and stores 16-bit values in pairs.
// 16384 rows of 4095 fp32 into bf16: 107 us value by value, 54 so (4096: 41).
template <typename TI, typename TO, bool kTokens64>
__global__ void __launch_bounds__(kLookupThreads) EmbeddingRaggedKernel(const void* __restrict__ tokens, const TI* __restrict__ weight, TO* __restrict__ out,
                                                                        uint64_t num_tokens, uint32_t parts, uint64_t rows, uint64_t width, float scale) {
  constexpr int kBytes = kLookupColumns * static_cast<int>(sizeof(TI)) + 16;
  __shared__ __align__(16) unsigned char memory[kLookupThreads / 32][kBytes];
  const int lane = threadIdx.x & 31;
  unsigned char* mine = memory[threadIdx.x / 32];
  const uint32_t block = blockIdx.x / parts, part = blockIdx.x - block * parts;
  const uint64_t t = static_cast<uint64_t>(block) * (kLookupThreads / 32) + threadIdx.x / 32;
  if (t >= num_tokens) return;
  const uint64_t first = static_cast<uint64_t>(part) * kLookupColumns;
  const int columns = static_cast<int>(min(width - first, static_cast<uint64_t>(kLookupColumns)));
  const int64_t id = Token<kTokens64>(tokens, t);
  const bool inside = id >= 0 && static_cast<uint64_t>(id) < rows;
  const uintptr_t begin = reinterpret_cast<uintptr_t>(weight + (inside ? static_cast<uint64_t>(id) : 0) * width + first);
  const TI* row = reinterpret_cast<const TI*>(mine + begin % 16);
  if (inside) {
    const unsigned to = static_cast<unsigned>(__cvta_generic_to_shared(mine));
    const uintptr_t end = begin + columns * sizeof(TI);
#pragma unroll
    for (int v = 0; v < kLookupColumns * static_cast<int>(sizeof(TI)) / 512 + 1; ++v) {
      const uintptr_t from = begin / 16 * 16 + (v * 32 + lane) * 16;
      if (from < end) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + (v * 32 + lane) * 16), "l"(from) : "memory");
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  __syncwarp();
  auto value = [&](int c) { return inside ? ToAcc<float, TI>(row[c]) * scale : 0.f; };
  TO* to = out + t * width + first;
  if constexpr (sizeof(TO) == 4) {
    for (int c = lane; c < columns; c += 32) to[c] = value(c);
  } else {
    const int head = reinterpret_cast<uintptr_t>(to) / 2 % 2;  // values before the first pair
    if (lane == 0 && head > 0) to[0] = FromAcc<TO, float>(value(0));
    const int pairs = (columns - head) / 2;
#pragma unroll 4
    for (int q = lane; q < pairs; q += 32) *reinterpret_cast<unsigned*>(to + head + 2 * q) = VecIO<TO>::P2(value(head + 2 * q), value(head + 2 * q + 1));
    if (lane == 0 && head + 2 * pairs < columns) to[columns - 1] = FromAcc<TO, float>(value(columns - 1));
  }
}

// The kernel behind may be set up while this one runs; it waits before it reads.
__device__ __forceinline__ void LetNextStart() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void WaitForPrevious() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// -------------------------------------------------------------------- sort
// The lanes of the warp with the same `bits` lowest bits of `d`, of those in `lanes`.
__device__ __forceinline__ unsigned Peers(unsigned lanes, uint32_t d, int bits) {
  unsigned peers = lanes;
  for (int b = 0; b < bits; ++b) {
    const bool set = d >> b & 1;
    const unsigned with = __ballot_sync(0xffffffffu, set);
    peers &= set ? with : ~with;
  }
  return peers;
}

constexpr int kSortThreads = 512;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMostDigitBits = 10;
constexpr int kMostSortBlocks = 64;
constexpr int kBatch = 4;  // elements of a thread that are loaded together

struct SortParams {
  const void* tokens;
  int tokens_are_64;
  uint32_t n;
  uint32_t rows;       // also the key of tokens without a gradient
  int64_t padding;
  uint32_t per_block;  // a multiple of kSortThreads
  int passes, bits;
  uint32_t* key[2];
  uint32_t* position[2];
  uint32_t* counts;    // gridDim.x x bins
  uint32_t* zeros;     // to be cleared for the kernel behind
  uint32_t num_zeros;
};

__device__ __forceinline__ uint32_t KeyOf(const SortParams& p, uint32_t t) {
  const int64_t id = p.tokens_are_64 ? Token<true>(p.tokens, t) : Token<false>(p.tokens, t);
  return id >= 0 && id < static_cast<int64_t>(p.rows) && id != p.padding ? static_cast<uint32_t>(id) : p.rows;
}

// A least-significant-digit radix sort, cooperative: a block's part of the list
// is cut into one part per warp, a digit's count of every warp gives the places.
// A warp places 32 elements at a time in their order, so every pass is stable.
// Equal digits in a warp are found by one ballot per bit (in the cluster's kernel
// as it was then, 16384 tokens, 14.1 us against 16.2 with `match.any`).  131072
// tokens of 32000 rows, two digits of 8 bits: 24 us by itself with cold caches, 22
// among the kernels of a call, where the next one is set up beside it.
__global__ void __launch_bounds__(kSortThreads) SortTokensKernel(SortParams p) {
  extern __shared__ uint32_t warp_counts[];  // kSortWarps x bins
  LetNextStart();
  __shared__ uint32_t scan[kSortWarps], bases[1 << kMostDigitBits];
  const cooperative_groups::grid_group grid = cooperative_groups::this_grid();
  const int bins = 1 << p.bits;
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const uint32_t part = p.per_block / kSortWarps;
  const uint32_t begin = blockIdx.x * p.per_block + warp * part;
  const uint32_t end = min(begin + part, p.n);
  uint32_t* mine = warp_counts + warp * bins;
  for (uint32_t i = blockIdx.x * kSortThreads + threadIdx.x; i < p.num_zeros; i += gridDim.x * kSortThreads) p.zeros[i] = 0;
  for (int pass = 0; pass < p.passes; ++pass) {
    const uint32_t* key_in = p.key[(pass + 1) & 1];
    const uint32_t* position_in = p.position[(pass + 1) & 1];
    uint32_t* key_out = p.key[pass & 1];
    uint32_t* position_out = p.position[pass & 1];
    const int shift = pass * p.bits;
    for (int i = threadIdx.x; i < kSortWarps * bins; i += kSortThreads) warp_counts[i] = 0;
    __syncthreads();
    for (uint32_t i0 = begin; i0 < end; i0 += 32 * kBatch) {
      uint32_t k[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const uint32_t i = i0 + u * 32 + lane;
        k[u] = i >= end ? 0 : pass == 0 ? KeyOf(p, i) : __ldcg(key_in + i);
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (i0 + u * 32 + lane < end) atomicAdd(&mine[(k[u] >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < bins; d += kSortThreads) {
      uint32_t sum = 0, c[kSortWarps];
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) c[w] = warp_counts[w * bins + d];
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) {
        warp_counts[w * bins + d] = sum;
        sum += c[w];
      }
      __stcg(p.counts + static_cast<size_t>(blockIdx.x) * bins + d, sum);
    }
    grid.sync();
    // Places of this block's elements of digit d: behind all smaller digits and behind digit d of the blocks before.
    uint32_t carried = 0;
    for (int d0 = 0; d0 < bins; d0 += kSortThreads) {
      const int d = d0 + threadIdx.x;
      uint32_t total = 0, before = 0;
      if (d < bins) {
#pragma unroll 32
        for (uint32_t g = 0; g < gridDim.x; ++g) {
          const uint32_t c = __ldcg(p.counts + static_cast<size_t>(g) * bins + d);
          before += g < blockIdx.x ? c : 0;
          total += c;
        }
      }
      uint32_t inclusive = total;
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, inclusive, s);
        if (lane >= s) inclusive += v;
      }
      if (lane == 31) scan[warp] = inclusive;
      __syncthreads();
      uint32_t base = carried, all = 0;
      for (int w = 0; w < kSortWarps; ++w) {
        base += w < warp ? scan[w] : 0;
        all += scan[w];
      }
      carried += all;
      if (d < bins) {
        bases[d] = base + inclusive - total + before;
      }
      __syncthreads();
    }
    for (uint32_t i0 = begin; i0 < end; i0 += 32 * kBatch) {
      uint32_t k[kBatch], at[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const uint32_t i = i0 + u * 32 + lane;
        k[u] = i >= end ? 0 : pass == 0 ? KeyOf(p, i) : __ldcg(key_in + i);
        at[u] = i >= end || pass == 0 ? i : __ldcg(position_in + i);
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const bool valid = i0 + u * 32 + lane < end;
        const uint32_t d = (k[u] >> shift) & (bins - 1);
        const unsigned peers = Peers(__ballot_sync(0xffffffffu, valid), d, p.bits);
        const uint32_t rank = mine[d] + __popc(peers & ((1u << lane) - 1));
        const uint32_t place = bases[d] + rank;
        __syncwarp();
        if (valid) {
          if (lane == 31 - __clz(peers)) mine[d] = rank + 1;
          __stcg(key_out + place, k[u]);
          __stcg(position_out + place, at[u]);
        }
        __syncwarp();
      }
    }
    if (pass + 1 < p.passes) grid.sync();
  }
}

// The same within one thread-block cluster, for lists that fit into its shared
// memory: a thread holds kItems elements in registers, counts go from block to
// block through distributed shared memory, elements are placed in the shared
// memory of the block that has them in the next pass.  Against the cooperative
// kernel, tokens of 50000 rows, by itself: 2048 8.5 us against 18.5, 16384 13 against 22,
// 32768 20.3 against 22.2, 65536 35 against 23 (there are only eight SMs to place
// the elements), so lists of up to 32768 are taken.
constexpr int kClusterThreads = 1024;
constexpr int kClusterWarps = kClusterThreads / 32;
constexpr int kClusterBlocks = 8;  // at most
constexpr int kMostItems = 4;

template <int kItems>
__global__ void __launch_bounds__(kClusterThreads) ClusterSortKernel(SortParams p) {
  extern __shared__ __align__(16) unsigned char memory[];
  const cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
  const uint32_t blocks = cluster.num_blocks();
  LetNextStart();
  constexpr uint32_t kPerBlock = kItems * kClusterThreads;
  const int bins = 1 << p.bits;
  uint2* elements = reinterpret_cast<uint2*>(memory);                                       // kPerBlock
  uint32_t* totals = reinterpret_cast<uint32_t*>(memory + kPerBlock * sizeof(uint2));       // bins
  uint32_t* bases = totals + bins;                                                          // bins
  unsigned short* counts = reinterpret_cast<unsigned short*>(bases + bins);                 // kClusterWarps x bins
  __shared__ uint32_t scan[kClusterWarps];
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  unsigned short* mine = counts + warp * bins;
  for (uint32_t i = blockIdx.x * kClusterThreads + threadIdx.x; i < p.num_zeros; i += blocks * kClusterThreads) p.zeros[i] = 0;
  for (int pass = 0; pass < p.passes; ++pass) {
    const int shift = pass * p.bits;
    uint32_t key[kItems], position[kItems], rank[kItems];
    const uint32_t first = warp * (32 * kItems) + lane;  // in the block; a warp's elements are adjacent
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const uint32_t at = first + i * 32, t = blockIdx.x * kPerBlock + at;
      if (pass == 0) {
        key[i] = t < p.n ? KeyOf(p, t) : 0;
        position[i] = t;
      } else {
        const uint2 e = elements[at];
        key[i] = e.x;
        position[i] = e.y;
      }
    }
    for (int i = threadIdx.x; i < kClusterWarps * bins / 2; i += kClusterThreads) reinterpret_cast<uint32_t*>(counts)[i] = 0;
    __syncthreads();
    // A place among the warp's elements of the same digit, in their order.
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const bool valid = blockIdx.x * kPerBlock + first + i * 32 < p.n;
      const uint32_t d = (key[i] >> shift) & (bins - 1);
      const unsigned peers = Peers(__ballot_sync(0xffffffffu, valid), d, p.bits);
      rank[i] = valid ? mine[d] + __popc(peers & ((1u << lane) - 1)) : 0;
      __syncwarp();
      if (valid && lane == 31 - __clz(peers)) mine[d] = static_cast<unsigned short>(rank[i] + 1);
      __syncwarp();
    }
    __syncthreads();
    // Of every digit, what the warps before have and what the block has.
    if (static_cast<int>(threadIdx.x) < bins) {
      uint32_t sum = 0, c[kClusterWarps];
#pragma unroll
      for (int w = 0; w < kClusterWarps; ++w) c[w] = counts[w * bins + threadIdx.x];
#pragma unroll
      for (int w = 0; w < kClusterWarps; ++w) {
        counts[w * bins + threadIdx.x] = static_cast<unsigned short>(sum);
        sum += c[w];
      }
      totals[threadIdx.x] = sum;
    }
    cluster.sync();  // the totals are there, and all elements are in registers
    uint32_t before = 0, all = 0;
    if (static_cast<int>(threadIdx.x) < bins) {
#pragma unroll
      for (int b = 0; b < kClusterBlocks; ++b) {
        const uint32_t c = b < static_cast<int>(blocks) ? *cluster.map_shared_rank(totals + threadIdx.x, b) : 0;
        before += b < static_cast<int>(blockIdx.x) ? c : 0;
        all += c;
      }
    }
    uint32_t inclusive = all;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, inclusive, s);
      if (lane >= s) inclusive += v;
    }
    if (lane == 31) scan[warp] = inclusive;
    __syncthreads();
    uint32_t smaller = scan[lane];  // kClusterWarps is 32
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, smaller, s);
      if (lane >= s) smaller += v;
    }
    smaller = __shfl_sync(0xffffffffu, smaller, (warp + 31) & 31);
    if (static_cast<int>(threadIdx.x) < bins) bases[threadIdx.x] = (warp > 0 ? smaller : 0) + inclusive - all + before;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      if (blockIdx.x * kPerBlock + first + i * 32 < p.n) {
        const uint32_t d = (key[i] >> shift) & (bins - 1);
        const uint32_t place = bases[d] + mine[d] + rank[i];
        *cluster.map_shared_rank(elements + place % kPerBlock, place / kPerBlock) = make_uint2(key[i], position[i]);
      }
    }
    cluster.sync();  // the elements are there, and nobody reads this block's totals any more
  }
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const uint32_t at = i * kClusterThreads + threadIdx.x, place = blockIdx.x * kPerBlock + at;
    if (place < p.n) {
      const uint2 e = elements[at];
      p.key[0][place] = e.x;
      p.position[0][place] = e.y;
    }
  }
}

// ------------------------------------------------------------------- clear
constexpr int kClearThreads = 256, kClearUnroll = 4;
constexpr uint64_t kClearBytes = static_cast<uint64_t>(kClearThreads) * kClearUnroll * 32;  // of a block

// out = 0.  It reads nothing, so it runs beside the sort, on the SMs that the sort
// leaves; its last block waits for the sort, so that whoever waits for this kernel
// has waited for both.  A table of 100003 x 2048 bf16: 56 us, 7.3 TB/s.
__global__ void __launch_bounds__(kClearThreads) ClearKernel(unsigned char* out, uint64_t bytes) {
  LetNextStart();
  const uint64_t head = min(static_cast<uint64_t>((32 - reinterpret_cast<uintptr_t>(out) % 32) % 32), bytes);
  const uint64_t quanta = (bytes - head) / 32;
  const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int u = 0; u < kClearUnroll; ++u) {
    const uint64_t q = (static_cast<uint64_t>(blockIdx.x) * kClearUnroll + u) * kClearThreads + threadIdx.x;
    if (q < quanta) St32(out + head + q * 32, zero, zero);
  }
  if (blockIdx.x == 0) {
    const uint64_t tail = head + quanta * 32;
    if (threadIdx.x < head) out[threadIdx.x] = 0;
    if (threadIdx.x < bytes - tail) out[tail + threadIdx.x] = 0;
  }
  if (blockIdx.x == gridDim.x - 1) WaitForPrevious();
}

// -------------------------------------------------------------------- sums
constexpr int kSumWarps = 8;
constexpr int kSumThreads = 32 * kSumWarps;
constexpr int kWarpTokens = 16;  // with 8 or 32, 16384 rows of 4096 take 82 or 77 us instead of 75
constexpr uint32_t kNoKey = 0xffffffffu;

struct SumParams {
  const uint32_t* key;
  const uint32_t* position;
  uint32_t n;
  uint32_t rows;
  uint32_t per_warp;  // tokens: 32 at most, or a multiple of 32
  uint32_t ranges;    // of kSumWarps * per_warp tokens
  uint32_t tiles;     // slices of the columns
  const void* grad;
  void* out;
  float* partial;     // [2 * ranges][width]: a range's run that began before it, the one that goes on behind it
  uint32_t* arrived;  // [ranges][tiles], zero
  uint64_t width;
  float scale;
  int accumulate;
};

// A warp's slice of a row: 256 columns, eight per lane: with kVector in vectors
// of at most 16 bytes of either type (a warp's access is one stretch of memory in
// both: with 32 bytes of fp32 per lane 16384 bf16 rows of 4096 took 67 us instead
// of 57), else one by one.  Rows come through a ring in shared memory, 4 KiB per
// warp and 128 KiB per SM; in registers the same bytes left room for three blocks
// per SM instead of four, and 131072 fp32 rows of 1024 took 180 us instead of 130.
// kOld: 16-bit tables that are added to; what a row holds comes with the gradient of
// the token that completes it.
template <typename TG, typename TO, bool kVector, bool kOld>
struct Slice {
  static constexpr int kCols = 8;
  static constexpr int kPer = !kVector ? 1 : sizeof(TG) == 2 && sizeof(TO) == 2 ? 8 : 4;  // adjacent columns
  static constexpr int kVecs = kCols / kPer;
  static constexpr int kRowBytes = 32 * kCols * static_cast<int>(sizeof(TG));
  static constexpr int kGradBytes = kRowBytes + (kVector ? 0 : 16);
  static constexpr int kOldBytes = !kOld ? 0 : 32 * kCols * static_cast<int>(sizeof(TO)) + (kVector ? 0 : 16);
  static constexpr int kSlotBytes = kGradBytes + kOldBytes;
  static constexpr int kSlots = kOld ? 4 : 4096 / kRowBytes;  // rows on their way to a warp
  static constexpr int kRing = kSumWarps * kSlots * kSlotBytes;
  uint64_t width;
  uint64_t column;  // the lane's first; the others are 32 * kPer apart
  __device__ __forceinline__ Slice(uint32_t tile, uint64_t w) : width(w), column(static_cast<uint64_t>(tile) * (32 * kCols) + (threadIdx.x & 31) * kPer) {}
  // With kVector the width is a multiple of kPer: a lane has all columns of a vector or none.
  __device__ __forceinline__ bool Has(int v) const { return column + v * (32 * kPer) < width; }

  // A row into one of the warp's slots (`slot`: its start), without waiting for it.  With kVector a lane copies what it
  // reads itself.  Else the warp copies the 16-byte words of memory that hold the slice: no allocation ends inside one,
  // and a row may start at any element of one.
  template <typename T>
  __device__ __forceinline__ void Fetch(const T* row, unsigned slot) const {
    constexpr int kBytes = kPer * static_cast<int>(sizeof(T));
    const int lane = threadIdx.x & 31;
    if constexpr (kVector) {
#pragma unroll
      for (int v = 0; v < kVecs; ++v) {
        if (Has(v)) {
          const T* from = row + column + v * (32 * kPer);
          const unsigned to = slot + (v * 32 + lane) * kBytes;
          if constexpr (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
          else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(from) : "memory");
        }
      }
    } else {
      const uint64_t first = column - lane, columns = min(width - first, static_cast<uint64_t>(32 * kCols));
      const uintptr_t begin = reinterpret_cast<uintptr_t>(row + first), end = begin + columns * sizeof(T);
#pragma unroll
      for (int v = 0; v < 32 * kCols * static_cast<int>(sizeof(T)) / 512 + 1; ++v) {
        const uintptr_t from = begin / 16 * 16 + (v * 32 + lane) * 16;
        if (from < end) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(slot + (v * 32 + lane) * 16), "l"(from) : "memory");
      }
    }
  }
  // sum += what Fetch has brought of `row`.
  template <typename T>
  __device__ __forceinline__ void AddSlot(const T* row, const unsigned char* slot, float* sum) const {
    constexpr int kBytes = kPer * static_cast<int>(sizeof(T));
    const int lane = threadIdx.x & 31;
    const unsigned char* at = slot + lane * kBytes;
    if constexpr (!kVector) at += reinterpret_cast<uintptr_t>(row + (column - lane)) % 16;
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      if constexpr (kBytes == 16) {
        VecIO<T>::Add(*reinterpret_cast<const uint4*>(at + v * 512), sum + v * kPer);
      } else if constexpr (kPer == 4) {
        const uint2 q = *reinterpret_cast<const uint2*>(at + v * 256);
        float a[8];
        VecIO<T>::Load(make_uint4(q.x, q.y, 0, 0), a);
#pragma unroll
        for (int e = 0; e < kPer; ++e) sum[v * kPer + e] += a[e];
      } else {
        if (Has(v)) sum[v] += ToAcc<float, T>(*reinterpret_cast<const T*>(at + v * 32 * sizeof(T)));
      }
    }
  }
  template <typename T>
  __device__ __forceinline__ void Load(const T* row, float* a) const {
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      if (Has(v)) {
        if constexpr (kVector) LoadValues<T, kPer>(row + column + v * (32 * kPer), a + v * kPer);
        else a[v] = ToAcc<float, T>(row[column + v * 32]);
      } else {
#pragma unroll
        for (int e = 0; e < kPer; ++e) a[v * kPer + e] = 0.f;
      }
    }
  }
  template <typename T>
  __device__ __forceinline__ void Store(T* row, const float* a) const {
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      if (Has(v)) {
        if constexpr (kVector) StoreValues<T, kPer>(row + column + v * (32 * kPer), a + v * kPer);
        else row[column + v * 32] = FromAcc<T, float>(a[v]);
      }
    }
  }
  // Added by the memory: nothing to wait for (16384 bf16 rows into fp32 75 us; loaded, added and stored 85).  Only one warp
  // adds to a row, once.  These additions take subnormal numbers (below 1.2e-38) for zero.
  __device__ __forceinline__ void Add(float* row, const float* a) const {
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      if (Has(v)) {
        float* at = row + column + v * (32 * kPer);
        if constexpr (kVector) {
#pragma unroll
          for (int e = 0; e < kPer; e += 4) {
            const float* b = a + v * kPer + e;
            asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(at + e), "f"(b[0]), "f"(b[1]), "f"(b[2]), "f"(b[3]) : "memory");
          }
        } else {
          atomicAdd(at, a[v]);
        }
      }
    }
  }
};

template <typename TO, typename S>
__device__ __forceinline__ void WriteRow(const SumParams& p, const S& slice, uint32_t row, const float* sum) {
  constexpr int kCols = S::kCols;
  TO* out = static_cast<TO*>(p.out) + static_cast<uint64_t>(row) * p.width;
  float v[kCols];
#pragma unroll
  for (int e = 0; e < kCols; ++e) v[e] = sum[e] * p.scale;
  if (!p.accumulate) {
    slice.Store(out, v);
  } else if constexpr (sizeof(TO) == 4) {
    slice.Add(out, v);
  } else {
    float old[kCols];
    slice.Load(out, old);
#pragma unroll
    for (int e = 0; e < kCols; ++e) v[e] += old[e];
    slice.Store(out, v);
  }
}

// The first and last range of the run of `k` that goes over an edge of `range`: a
// look at the 32 edges next to it, and a search in steps of a 32nd where the run
// goes over all of them.
__device__ __forceinline__ void RangesOfRun(const SumParams& p, uint32_t k, uint32_t range, uint32_t* first, uint32_t* last) {
  const uint32_t lane = threadIdx.x & 31, per = p.per_warp * kSumWarps;
  // Whether the run goes over edge b, which is that between range b - 1 and range b, if it goes over the next one, or the one before.
  auto from_left = [&](uint32_t b) { return b >= 1 && p.key[b * per - 1] == k; };
  auto to_right = [&](uint32_t b) { return b < p.ranges && p.key[b * per] == k; };
  const bool over_left = from_left(range) && to_right(range);
  unsigned m = __ballot_sync(0xffffffffu, over_left && range >= lane && from_left(range - lane));
  uint32_t c = range - (m == 0xffffffffu ? 32 : __ffs(~m) - 1);  // the run goes over the edges c + 1 to range
  if (m == 0xffffffffu) {
    uint32_t lo = 0, hi = c + 1;  // not over edge lo, over edge hi
    while (hi - lo > 1) {
      const uint32_t step = (hi - lo + 31) / 32, b = lo + step * (lane + 1);
      const int f = __ffs(__ballot_sync(0xffffffffu, b >= hi || from_left(b))) - 1;
      hi = min(hi, lo + step * (f + 1));
      lo += step * f;
    }
    c = hi - 1;
  }
  *first = c;
  m = __ballot_sync(0xffffffffu, range + 1 < p.ranges && from_left(range + 1) && to_right(range + 1 + lane));
  c = range + (m == 0xffffffffu ? 32 : __ffs(~m) - 1);  // over the edges range + 1 to c
  if (m == 0xffffffffu) {
    uint32_t lo = c, hi = p.ranges;  // over edge lo, not over edge hi
    while (hi - lo > 1) {
      const uint32_t step = (hi - lo + 31) / 32, b = lo + step * (lane + 1);
      const int f = __ffs(__ballot_sync(0xffffffffu, b >= hi || !to_right(b))) - 1;
      hi = min(hi, lo + step * (f + 1));
      lo += step * f;
    }
    c = lo;
  }
  *last = c;
}

// A block adds the rows of a range of the sorted tokens, in a slice of the
// columns; a warp takes a part of the range.  Runs inside a warp's part are
// written at once, those over the edges of parts are joined through shared
// memory, those over the edges of the range through the workspace by the block
// that comes last: always in the tokens' order.  `ring`: S::kRing bytes.
template <typename TG, typename TO, bool kVector, bool kOld>
__device__ __forceinline__ void SumRange(const SumParams& p, uint32_t range, uint32_t tile, unsigned char* ring) {
  using S = Slice<TG, TO, kVector, kOld>;
  constexpr int kCols = S::kCols;
  __shared__ float part[kSumWarps][2][32 * kCols];  // runs that began before the part, that go on behind it
  __shared__ uint32_t before_key[kSumWarps], first_key[kSumWarps], last_key[kSumWarps], behind_key[kSumWarps];
  __shared__ uint32_t run_first[2], run_last[2], is_last[2];  // of the runs over the range's two edges
  const S slice(tile, p.width);
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const uint32_t i0 = (range * kSumWarps + warp) * p.per_warp;
  const int count = i0 < p.n ? static_cast<int>(min(p.per_warp, p.n - i0)) : 0;
  const uint32_t before = count > 0 && i0 > 0 ? p.key[i0 - 1] : kNoKey;
  const uint32_t last = count > 0 ? p.key[i0 + count - 1] : kNoKey;
  const uint32_t behind = count > 0 && i0 + count < p.n ? p.key[i0 + count] : kNoKey;
  const TG* grad = static_cast<const TG*>(p.grad);
  float sum[kCols];
#pragma unroll
  for (int e = 0; e < kCols; ++e) sum[e] = 0.f;
  // 32 tokens of the part, a lane holds one.
  struct Held {
    uint32_t key, position;
    int known;      // those with a row, which come first
    unsigned ends;  // those that end a run, or the part
  };
  auto hold = [&](int at) {
    Held h;
    const int n = min(max(count - at, 0), 32);
    h.key = lane < n ? p.key[i0 + at + lane] : kNoKey;
    h.position = lane < n ? p.position[i0 + at + lane] : 0;
    const uint32_t after = n > 0 && i0 + at + n < p.n ? p.key[i0 + at + n] : kNoKey;
    uint32_t next = __shfl_down_sync(0xffffffffu, h.key, 1);
    if (lane == n - 1) next = at + n == count ? kNoKey : after;
    h.known = __popc(__ballot_sync(0xffffffffu, h.key < p.rows));
    h.ends = __ballot_sync(0xffffffffu, lane < h.known && h.key != next);
    return h;
  };
  Held held = hold(0), ahead = hold(32);
  // Whether the first and the last run go over the part's edges.
  const uint32_t begin_key = __shfl_sync(0xffffffffu, held.key, 0);
  const bool began_before = begin_key < p.rows && before == begin_key;
  const bool goes_on = last < p.rows && behind == last;
  bool first = true;  // no run of the part has ended
  auto table = [&](uint32_t k) { return static_cast<TO*>(p.out) + static_cast<uint64_t>(k) * p.width; };
  // The run that token j of the part, of row k, ends is complete.
  auto flush = [&](int j, uint32_t k, const unsigned char* old) {
    const bool head = first && began_before;
    if (head || (goes_on && j == count - 1)) {
      float* mine = part[warp][head ? 0 : 1];
#pragma unroll
      for (int e = 0; e < kCols; ++e) mine[e * 32 + lane] = sum[e];
    } else if constexpr (kOld) {
      TO* to = table(k);
#pragma unroll
      for (int e = 0; e < kCols; ++e) sum[e] *= p.scale;
      slice.AddSlot(to, old, sum);
      slice.Store(to, sum);
    } else {
      WriteRow<TO>(p, slice, k, sum);
    }
    first = false;
#pragma unroll
    for (int e = 0; e < kCols; ++e) sum[e] = 0.f;
  };
  auto row = [&](const Held& h, int j) { return grad + static_cast<uint64_t>(__shfl_sync(0xffffffffu, h.position, j)) * p.width; };
  // How far the runs over the range's edges reach, looked up while the first rows are on their way.
  auto reach = [&](int side, uint32_t k) {
    uint32_t a, b;
    RangesOfRun(p, k, range, &a, &b);
    if (lane == 0) run_first[side] = a, run_last[side] = b;
  };
  constexpr int kSlot = S::kSlotBytes;
  unsigned char* mine = ring + warp * (S::kSlots * kSlot);
  const unsigned mine_shared = static_cast<unsigned>(__cvta_generic_to_shared(mine));
  auto fetch = [&](const Held& h, int j, int u) {
    const TG* r = row(h, j);
    const uint32_t k = kOld ? __shfl_sync(0xffffffffu, h.key, j) : 0;
    if (j < h.known) {
      slice.Fetch(r, mine_shared + u * kSlot);
      if constexpr (kOld)
        if (h.ends >> j & 1) slice.Fetch(static_cast<const TO*>(table(k)), mine_shared + u * kSlot + S::kGradBytes);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int u = 0; u < S::kSlots; ++u) fetch(held, u, u);
  if (warp == 0 && began_before) reach(0, begin_key);
  if (warp == kSumWarps - 1 && goes_on) reach(1, last);
  for (int at = 0; at < count; at += 32) {
    for (int j0 = 0; j0 < held.known; j0 += S::kSlots) {
#pragma unroll
      for (int u = 0; u < S::kSlots; ++u) {
        const int j = j0 + u;
        if (j < held.known) {
          asm volatile("cp.async.wait_group %0;" ::"n"(S::kSlots - 1) : "memory");
          if constexpr (!kVector) __syncwarp();  // what the other lanes have copied
          slice.AddSlot(row(held, j), mine + u * kSlot, sum);
          // With kOld the slot is needed for the flush; else the next row is sent for first.
          if constexpr (kOld)
            if (held.ends >> j & 1) flush(at + j, __shfl_sync(0xffffffffu, held.key, j), mine + u * kSlot + S::kGradBytes);
          if constexpr (!kVector) __syncwarp();  // they have read it
          if (j + S::kSlots < 32) fetch(held, j + S::kSlots, u);
          else fetch(ahead, j + S::kSlots - 32, u);
          if constexpr (!kOld)
            if (held.ends >> j & 1) flush(at + j, __shfl_sync(0xffffffffu, held.key, j), nullptr);
        }
      }
    }
    held = ahead;
    ahead = hold(at + 64);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if (lane == 0) {
    before_key[warp] = before;
    first_key[warp] = begin_key;
    last_key[warp] = last;
    behind_key[warp] = behind;
  }
  __syncthreads();
  // Runs over the edges of parts.
  const bool from_before = first_key[0] < p.rows && before_key[0] == first_key[0];
  auto join = [&](int w, bool head) {
    const uint32_t k = head ? first_key[w] : last_key[w];
    bool on = last_key[w] == k && behind_key[w] == k;
#pragma unroll
    for (int e = 0; e < kCols; ++e) sum[e] = part[w][head ? 0 : 1][e * 32 + lane];
    while (on && ++w < kSumWarps) {
#pragma unroll
      for (int e = 0; e < kCols; ++e) sum[e] += part[w][0][e * 32 + lane];
      on = last_key[w] == k && behind_key[w] == k;
    }
    if (head || on) slice.Store(p.partial + (2 * static_cast<uint64_t>(range) + (head ? 0 : 1)) * p.width, sum);
    else WriteRow<TO>(p, slice, k, sum);
  };
  if (warp == 0 && from_before) join(0, true);
  const uint32_t k = last_key[warp];
  if (k < p.rows && behind_key[warp] == k && !(first_key[warp] == k && before_key[warp] == k)) join(warp, false);
  // Runs over the edges of the range.
  const uint32_t end = last_key[kSumWarps - 1];
  const bool to_behind = end < p.rows && behind_key[kSumWarps - 1] == end && !(from_before && first_key[0] == end);
  if (!from_before && !to_behind) return;
  __syncthreads();
  if (threadIdx.x < 2 && (threadIdx.x == 0 ? from_before : to_behind)) {
    __threadfence();  // the block's parts are there before it counts as arrived
    const uint32_t a = run_first[threadIdx.x];
    is_last[threadIdx.x] = atomicAdd(p.arrived + static_cast<uint64_t>(a) * p.tiles + tile, 1u) == run_last[threadIdx.x] - a;
    __threadfence();
  }
  __syncthreads();
  for (int side = from_before ? 0 : 1; side < (to_behind ? 2 : 1); ++side) {
    if (!is_last[side]) continue;
    const uint32_t row = side == 0 ? first_key[0] : end;
    const uint32_t parts = run_last[side] - run_first[side] + 1;
    const uint32_t begin = static_cast<uint32_t>(static_cast<uint64_t>(parts) * warp / kSumWarps);
    const uint32_t stop = static_cast<uint32_t>(static_cast<uint64_t>(parts) * (warp + 1) / kSumWarps);
#pragma unroll
    for (int e = 0; e < kCols; ++e) sum[e] = 0.f;
#pragma unroll 4
    for (uint32_t i = begin; i < stop; ++i) {
      float a[kCols];
      // The run goes on behind its first range and began before the others.
      slice.Load(p.partial + (2 * static_cast<uint64_t>(run_first[side] + i) + (i == 0 ? 1 : 0)) * p.width, a);
#pragma unroll
      for (int e = 0; e < kCols; ++e) sum[e] += a[e];
    }
#pragma unroll
    for (int e = 0; e < kCols; ++e) part[warp][0][e * 32 + lane] = sum[e];
    __syncthreads();
    if (warp == 0) {
      for (int w = 1; w < kSumWarps; ++w) {
#pragma unroll
        for (int e = 0; e < kCols; ++e) sum[e] += part[w][0][e * 32 + lane];
      }
      WriteRow<TO>(p, slice, row, sum);
    }
    __syncthreads();
  }
}

template <typename TG, typename TO, bool kVector, bool kOld>
__global__ void __launch_bounds__(kSumThreads, 4) SumRunsKernel(SumParams p) {
  extern __shared__ __align__(16) unsigned char ring[];
  WaitForPrevious();
  const uint32_t range = blockIdx.x / p.tiles;
  SumRange<TG, TO, kVector, kOld>(p, range, blockIdx.x - range * p.tiles, ring);
}

// Few tokens: every block sorts them all, by counting for each how many come
// before it, and adds the runs that begin in its part of the list, in its slice
// of the columns.  The blocks behind clear rows that no token names.  One launch:
// 33 rows of 768 bf16 3.3 us on the device against 11 with the kernels above, 256
// rows 5.7 against 11.1 (11.1 too with one part for all).  More tokens than threads are not taken: a block
// would count for n * n / 256 pairs.
constexpr uint32_t kSmallTokens = kSumThreads;
constexpr uint32_t kPartTokens = 32;  // of a block: four per warp
constexpr uint32_t kClearRows = 8192;  // of a block, at most

struct SmallParams {
  SumParams sum;  // key and position are the block's own
  const void* tokens;
  int tokens_are_64;
  int64_t padding;
  uint32_t parts;       // of the list, a block per part and slice
  uint32_t clear_rows;  // of a block
};

template <typename TG, typename TO, bool kVector, bool kOld>
__global__ void __launch_bounds__(kSumThreads, 4) FewTokensKernel(SmallParams p) {
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ __align__(16) uint32_t keys[kSmallTokens], sorted[kSmallTokens], positions[kSmallTokens], named[kClearRows / 32], bounds[2];
  const uint32_t t = threadIdx.x, n = p.sum.n;
  SortParams of{};
  of.tokens = p.tokens;
  of.tokens_are_64 = p.tokens_are_64;
  of.rows = p.sum.rows;
  of.padding = p.padding;
  const uint32_t key = t < n ? KeyOf(of, t) : kNoKey;
  if (blockIdx.x < p.sum.tiles * p.parts) {
    keys[t] = key;
    __syncthreads();
    uint32_t rank = 0;
    const uint4* four = reinterpret_cast<const uint4*>(keys);
    for (uint32_t j = 0; j < n; j += 4) {
      const uint4 k = four[j / 4];
      rank += (k.x < key + (j < t)) + (k.y < key + (j + 1 < t)) + (k.z < key + (j + 2 < t)) + (k.w < key + (j + 3 < t));
    }
    if (t < n) {
      sorted[rank] = key;
      positions[rank] = t;
    }
    if (t < 2) bounds[t] = n;
    __syncthreads();
    // The block's share: from the first run that begins in its part of the list to the first that begins behind it.
    const uint32_t part = blockIdx.x / p.sum.tiles, lo = part * n / p.parts, hi = (part + 1) * n / p.parts;
    if (t < n && (t == 0 || sorted[t] != sorted[t - 1])) {
      if (t >= lo) atomicMin(&bounds[0], t);
      if (t >= hi) atomicMin(&bounds[1], t);
    }
    __syncthreads();
    SumParams sum = p.sum;
    sum.key = sorted + bounds[0];
    sum.position = positions + bounds[0];
    sum.n = bounds[1] - bounds[0];
    sum.per_warp = (sum.n + kSumWarps - 1) / kSumWarps;
    if (sum.n > 0) SumRange<TG, TO, kVector, kOld>(sum, 0, blockIdx.x - part * p.sum.tiles, ring);
    return;
  }
  const uint32_t first = (blockIdx.x - p.sum.tiles * p.parts) * p.clear_rows, rows = min(p.clear_rows, p.sum.rows - first);
  for (uint32_t i = t; i < kClearRows / 32; i += kSumThreads) named[i] = 0;
  __syncthreads();
  if (key >= first && key - first < rows) atomicOr(&named[(key - first) / 32], 1u << (key - first) % 32);
  __syncthreads();
  // Stores of 16 bytes where a row is made of them.
  constexpr uint32_t kPer = kVector ? 16 / sizeof(TO) : 1;
  const uint32_t width = static_cast<uint32_t>(p.sum.width);
  TO* out = static_cast<TO*>(p.sum.out) + static_cast<uint64_t>(first) * width;
  const bool wide = kVector && width % kPer == 0 && reinterpret_cast<uintptr_t>(p.sum.out) % 16 == 0;
  const uint32_t per_row = wide ? width / kPer : width;
  const uint64_t units = static_cast<uint64_t>(rows) * per_row;
  for (uint64_t u = t; u < units; u += kSumThreads) {
    const uint32_t row = static_cast<uint32_t>(u / per_row);
    if (named[row / 32] >> row % 32 & 1) continue;
    if (wide) St16(out + u * kPer, make_uint4(0, 0, 0, 0));
    else out[u] = FromAcc<TO, float>(0.f);
  }
}

}  // namespace dev

namespace {

template <typename TI, typename TO, bool kTokens64>
cudaError_t LaunchLookup(const EmbeddingParams& p, cudaStream_t stream) {
  constexpr int kN = dev::LookupQuantum<TI, TO>::kN;
  auto aligned = [](const void* a, size_t bytes) { return reinterpret_cast<uintptr_t>(a) % std::min<size_t>(bytes, 16) == 0; };
  const bool vector = p.width % kN == 0 && aligned(p.weight, kN * sizeof(TI)) && aligned(p.out, kN * sizeof(TO));
  const TI* w = static_cast<const TI*>(p.weight);
  TO* o = static_cast<TO*>(p.out);
  const float scale = static_cast<float>(p.scale);
  int lanes = 0;
  if (vector)
    while (lanes < 5 && (1ull << lanes) < p.width / kN) ++lanes;
  else lanes = 5;
  const uint64_t per_block = static_cast<uint64_t>(dev::kLookupThreads) >> lanes;
  const uint64_t blocks = (p.num_tokens + per_block - 1) / per_block;
  const uint64_t columns = vector ? (static_cast<uint64_t>(dev::kLookupUnroll) << lanes) * kN : dev::kLookupColumns;
  const uint64_t parts = (p.width + columns - 1) / columns;
  if (blocks * parts > 0x7fffffffull) return cudaErrorInvalidValue;
  const unsigned grid = static_cast<unsigned>(blocks * parts);
  if (vector) {
    dev::EmbeddingKernel<TI, TO, kTokens64><<<grid, dev::kLookupThreads, 0, stream>>>(p.tokens, w, o, p.num_tokens, static_cast<uint32_t>(p.width / kN),
                                                                                     static_cast<uint32_t>(parts), lanes, p.rows, p.width, scale);
  } else {
    dev::EmbeddingRaggedKernel<TI, TO, kTokens64><<<grid, dev::kLookupThreads, 0, stream>>>(p.tokens, w, o, p.num_tokens, static_cast<uint32_t>(parts), p.rows,
                                                                                           p.width, scale);
  }
  return cudaGetLastError();
}

// f(TI{}, TO{}) for a pair of the floating types that the embedding takes.
template <typename TI, typename F>
cudaError_t WithOutput(int dtype, F f) {
  switch (static_cast<DType>(dtype)) {
    case DType::kFloat32: return f(TI{}, float{});
    case DType::kFloat16: return f(TI{}, __half{});
    case DType::kBFloat16: return f(TI{}, __nv_bfloat16{});
    default: return cudaErrorInvalidValue;
  }
}
template <typename F>
cudaError_t WithTypes(int dtype_in, int dtype_out, F f) {
  switch (static_cast<DType>(dtype_in)) {
    case DType::kFloat32: return WithOutput<float>(dtype_out, f);
    case DType::kFloat16: return WithOutput<__half>(dtype_out, f);
    case DType::kBFloat16: return WithOutput<__nv_bfloat16>(dtype_out, f);
    default: return cudaErrorInvalidValue;
  }
}

struct SortShape {
  int passes, bits, blocks;
  uint32_t per_block;
  int items;  // per thread of a cluster's blocks; 0: the cooperative kernel
};
// The list in s->blocks parts for the cooperative kernel, or fewer where that many are not needed.
void CutSort(uint64_t n, SortShape* s) {
  uint64_t per = (n + s->blocks - 1) / s->blocks;
  per = std::max<uint64_t>((per + dev::kSortThreads - 1) / dev::kSortThreads, 1) * dev::kSortThreads;
  s->per_block = static_cast<uint32_t>(per);
  s->blocks = static_cast<int>((n + per - 1) / per);
}
SortShape ShapeOf(uint64_t n, uint64_t rows) {
  SortShape s;
  int all = 1;  // bits of the keys, 0 .. rows
  while (all < 32 && (rows >> all) != 0) ++all;
  s.passes = (all + dev::kMostDigitBits - 1) / dev::kMostDigitBits;
  s.bits = (all + s.passes - 1) / s.passes;
  // In a cluster, as few blocks and elements per thread as hold the list.
  s.items = 0;
  if (n <= static_cast<uint64_t>(dev::kClusterBlocks) * dev::kMostItems * dev::kClusterThreads) {
    s.blocks = 1;
    s.items = 1;
    while (s.blocks < dev::kClusterBlocks && static_cast<uint64_t>(s.blocks) * dev::kClusterThreads < n) s.blocks *= 2;
    while (static_cast<uint64_t>(s.blocks) * s.items * dev::kClusterThreads < n) s.items *= 2;
    s.per_block = 0;
    return s;
  }
  // A block takes at least 2048 tokens: with fewer the blocks' counts cost more than the tokens.
  s.blocks = static_cast<int>(std::min<uint64_t>(std::max<uint64_t>((n + 2047) / 2048, 1), dev::kMostSortBlocks));
  CutSort(n, &s);
  return s;
}

size_t Padded(size_t bytes) { return (bytes + 255) / 256 * 256; }

constexpr uint64_t kFewClearBytes = 128 << 10;  // of a block that looks for the rows of few tokens

// A launch that may be set up while the one before it in the stream runs.
template <typename... Params, typename... Args>
cudaError_t LaunchEarly(void (*kernel)(Params...), unsigned blocks, int threads, size_t smem, cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(blocks);
  config.blockDim = dim3(static_cast<unsigned>(threads));
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, args...);
}

// Shared memory of the sorts, which depends on the table's rows.  What a kernel is
// allowed belongs to all threads of the process: it is always what the largest
// table needs, so that no call takes from another one that is about to launch.
constexpr size_t ClusterSortBytes(int items, int bits) {
  return static_cast<size_t>(items) * dev::kClusterThreads * sizeof(uint2) + ((8 + dev::kClusterWarps * 2ull) << bits);
}
constexpr size_t SortBytes(int bits) { return (dev::kSortWarps * 4ull) << bits; }

template <int kItems>
cudaError_t LaunchClusterSort(const dev::SortParams& sort, const SortShape& shape, cudaStream_t stream) {
  const size_t smem = ClusterSortBytes(kItems, shape.bits);
  auto kernel = dev::ClusterSortKernel<kItems>;
  cudaError_t e = AllowSharedMemory(kernel, ClusterSortBytes(kItems, dev::kMostDigitBits));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(shape.blocks));
  config.blockDim = dim3(dev::kClusterThreads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = static_cast<unsigned>(shape.blocks);
  attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, sort);
}

}  // namespace

cudaError_t LaunchEmbedding(const EmbeddingParams& p, cudaStream_t stream) {
  if (p.num_tokens == 0 || p.width == 0) return cudaSuccess;
  return WithTypes(p.dtype_weight, p.dtype_out, [&](auto ti, auto to) {
    return p.tokens_are_64 ? LaunchLookup<decltype(ti), decltype(to), true>(p, stream) : LaunchLookup<decltype(ti), decltype(to), false>(p, stream);
  });
}

struct SumShape {
  uint32_t per_warp;
  uint64_t ranges, tiles;
};
SumShape SumShapeOf(uint64_t n, uint64_t rows, uint64_t width) {
  SumShape s;
  s.per_warp = n > dev::kSmallTokens ? dev::kWarpTokens : static_cast<uint32_t>((n + dev::kSumWarps - 1) / dev::kSumWarps);
  s.tiles = (width + 255) / 256;
  auto ranges = [&] { return (n + s.per_warp * dev::kSumWarps - 1) / (s.per_warp * dev::kSumWarps); };
  // Shorter parts where the blocks would not fill the GPU twice (148 SMs): their lengths are then what counts, not the runs over
  // their edges.  600 tokens of 768 13.5 -> 9.3 us, 8192 18.8 -> 17.9; 600 of 4096, skewed, 11.7 -> 12.7.
  if (n > dev::kSmallTokens)
    while (s.per_warp > 4 && ranges() * s.tiles < 2 * 148) s.per_warp /= 2;
  // Longer ones where the runs are long, at least on average, so that every range has one over each edge, as long as there are
  // two blocks per SM; 128 tokens only where there are eight.  Rows of bf16, 2 rows in the table: 32768 of 1024 33.7 us with 16
  // or 32, 27.2 with 64; 131072 of 1024 74.0 with 64, 74.8 with 128; 1 M of 512 527 with 16, 274 with 64, 260 with 128.
  if (n / std::max<uint64_t>(rows, 1) >= 8)
    while (s.per_warp < 128 && ranges() * s.tiles >= (s.per_warp < 64 ? 4 : 16) * 148) s.per_warp *= 2;
  s.ranges = n > 0 ? ranges() : 0;
  return s;
}

size_t EmbeddingGradWorkBytes(uint64_t n, uint64_t rows, uint64_t width) {
  if (n <= dev::kSmallTokens) return 0;
  const SortShape s = ShapeOf(n, rows);
  const SumShape sum = SumShapeOf(n, rows, width);
  return 4 * Padded(n * 4) + Padded(static_cast<size_t>(s.blocks) << s.bits << 2) + Padded(sum.ranges * sum.tiles * 4) + 2 * sum.ranges * width * 4;
}

// Sorts the tokens; `sum` gets what lies in the workspace.
static cudaError_t LaunchSort(const EmbeddingGradParams& p, dev::SumParams* sum, cudaStream_t stream) {
  SortShape shape = ShapeOf(p.num_tokens, p.rows);
  char* work = static_cast<char*>(p.work);
  auto take = [&](size_t bytes) {
    char* at = work;
    work += Padded(bytes);
    return at;
  };
  dev::SortParams sort{};
  sort.tokens = p.tokens;
  sort.tokens_are_64 = p.tokens_are_64;
  sort.n = sum->n;
  sort.rows = sum->rows;
  sort.padding = p.padding;
  sort.per_block = shape.per_block;
  sort.passes = shape.passes;
  sort.bits = shape.bits;
  for (int i = 0; i < 2; ++i) {
    sort.key[i] = reinterpret_cast<uint32_t*>(take(p.num_tokens * 4));
    sort.position[i] = reinterpret_cast<uint32_t*>(take(p.num_tokens * 4));
  }
  sort.counts = reinterpret_cast<uint32_t*>(take(static_cast<size_t>(shape.blocks) << shape.bits << 2));
  sort.num_zeros = sum->ranges * sum->tiles;
  sort.zeros = reinterpret_cast<uint32_t*>(take(static_cast<size_t>(sort.num_zeros) * 4));
  cudaError_t e = cudaSuccess;
  int last = 0;  // which of the two lists is the sorted one
  switch (shape.items) {
    case 1: e = LaunchClusterSort<1>(sort, shape, stream); break;
    case 2: e = LaunchClusterSort<2>(sort, shape, stream); break;
    case 4: e = LaunchClusterSort<4>(sort, shape, stream); break;
    default: {
      const size_t smem = SortBytes(shape.bits);
      e = AllowSharedMemory(dev::SortTokensKernel, SortBytes(dev::kMostDigitBits));
      if (e == cudaSuccess) e = LaunchTogether(dev::SortTokensKernel, shape.blocks, dev::kSortThreads, smem, stream, sort);
      while (e == cudaErrorCooperativeLaunchTooLarge && shape.blocks > 1) {
        shape.blocks /= 2;
        CutSort(p.num_tokens, &shape);
        sort.per_block = shape.per_block;
        e = LaunchTogether(dev::SortTokensKernel, shape.blocks, dev::kSortThreads, smem, stream, sort);
      }
      last = (shape.passes - 1) & 1;
    }
  }
  sum->key = sort.key[last];
  sum->position = sort.position[last];
  sum->arrived = sort.zeros;
  sum->partial = reinterpret_cast<float*>(work);
  return e;
}

cudaError_t LaunchEmbeddingGrad(const EmbeddingGradParams& p, cudaStream_t stream) {
  if (p.rows == 0 || p.width == 0) return cudaSuccess;
  if (p.num_tokens > 0x7fffffffull || p.rows > 0x7ffffffeull) return cudaErrorInvalidValue;
  const size_t size_out = static_cast<DType>(p.dtype_out) == DType::kFloat32 ? 4 : 2;
  const bool few = p.num_tokens > 0 && p.num_tokens <= dev::kSmallTokens;
  const uint64_t bytes = p.accumulate ? 0 : p.rows * p.width * size_out;
  const uint64_t clears = (bytes + dev::kClearBytes - 1) / dev::kClearBytes;
  if (clears > 0x7fffffffull) return cudaErrorInvalidValue;
  if (p.num_tokens == 0) {
    if (clears == 0) return cudaSuccess;
    dev::ClearKernel<<<static_cast<unsigned>(clears), dev::kClearThreads, 0, stream>>>(static_cast<unsigned char*>(p.out), bytes);
    return cudaGetLastError();
  }
  if (p.work_bytes < EmbeddingGradWorkBytes(p.num_tokens, p.rows, p.width)) return cudaErrorInvalidValue;
  const SumShape part = SumShapeOf(p.num_tokens, p.rows, p.width);
  if (part.ranges * part.tiles > 0x7fffffffull) return cudaErrorInvalidValue;
  dev::SumParams sum{};
  sum.n = static_cast<uint32_t>(p.num_tokens);
  sum.rows = static_cast<uint32_t>(p.rows);
  sum.per_warp = part.per_warp;
  sum.ranges = static_cast<uint32_t>(part.ranges);
  sum.tiles = static_cast<uint32_t>(part.tiles);
  sum.grad = p.grad;
  sum.out = p.out;
  sum.width = p.width;
  sum.scale = static_cast<float>(p.scale);
  sum.accumulate = p.accumulate ? 1 : 0;
  if (!few) {
    cudaError_t e = LaunchSort(p, &sum, stream);
    if (e == cudaSuccess && clears > 0)
      e = LaunchEarly(dev::ClearKernel, static_cast<unsigned>(clears), dev::kClearThreads, 0, stream, static_cast<unsigned char*>(p.out), bytes);
    if (e != cudaSuccess) return e;
  }
  return WithTypes(p.dtype_grad, p.dtype_out, [&](auto tg, auto to) {
    using TG = decltype(tg);
    using TO = decltype(to);
    constexpr uint64_t kPer = dev::Slice<TG, TO, true, false>::kPer;
    auto aligned = [](const void* a, size_t bytes) { return reinterpret_cast<uintptr_t>(a) % std::min<size_t>(bytes, 16) == 0; };
    const bool vector = p.width % kPer == 0 && aligned(p.grad, kPer * sizeof(TG)) && aligned(p.out, kPer * sizeof(TO));
    const unsigned grid = static_cast<unsigned>(part.ranges * part.tiles);
    if (few) {
      dev::SmallParams small{sum, p.tokens, p.tokens_are_64, p.padding, (sum.n + dev::kPartTokens - 1) / dev::kPartTokens, 0};
      const uint64_t row = p.width * sizeof(TO);
      small.clear_rows = static_cast<uint32_t>(std::min<uint64_t>(std::max<uint64_t>(kFewClearBytes / row, 1), dev::kClearRows));
      const uint64_t blocks = part.tiles * small.parts + (p.accumulate ? 0 : (p.rows + small.clear_rows - 1) / small.clear_rows);
      if (blocks > 0x7fffffffull) return cudaErrorInvalidValue;
      auto launch = [&](auto kernel, int ring) {
        const cudaError_t e = AllowSharedMemory(kernel, static_cast<size_t>(ring));
        if (e != cudaSuccess) return e;
        kernel<<<static_cast<unsigned>(blocks), dev::kSumThreads, ring, stream>>>(small);
        return cudaGetLastError();
      };
      if constexpr (sizeof(TO) == 2)
        if (p.accumulate) return vector ? launch(dev::FewTokensKernel<TG, TO, true, true>, dev::Slice<TG, TO, true, true>::kRing)
                                        : launch(dev::FewTokensKernel<TG, TO, false, true>, dev::Slice<TG, TO, false, true>::kRing);
      return vector ? launch(dev::FewTokensKernel<TG, TO, true, false>, dev::Slice<TG, TO, true, false>::kRing)
                    : launch(dev::FewTokensKernel<TG, TO, false, false>, dev::Slice<TG, TO, false, false>::kRing);
    }
    auto launch = [&](auto kernel, int ring) {
      const cudaError_t e = AllowSharedMemory(kernel, static_cast<size_t>(ring));
      if (e != cudaSuccess) return e;
      return LaunchEarly(kernel, grid, dev::kSumThreads, static_cast<size_t>(ring), stream, sum);
    };
    if constexpr (sizeof(TO) == 2)
      if (p.accumulate) return vector ? launch(dev::SumRunsKernel<TG, TO, true, true>, dev::Slice<TG, TO, true, true>::kRing)
                                      : launch(dev::SumRunsKernel<TG, TO, false, true>, dev::Slice<TG, TO, false, true>::kRing);
    return vector ? launch(dev::SumRunsKernel<TG, TO, true, false>, dev::Slice<TG, TO, true, false>::kRing)
                  : launch(dev::SumRunsKernel<TG, TO, false, false>, dev::Slice<TG, TO, false, false>::kRing);
  });
}

}  // namespace ibcomm
