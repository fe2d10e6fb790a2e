// The norm of a list of tensors taken as one vector, and clipping:
//   N = sqrt(sum x^2)  (or max |x|),   out = round(x * min(1, max_norm / (N + 1e-6))).
//
// The list travels in the kernel's parameters (nothing is copied ahead of the
// launch, and a captured call keeps its own).  Tensors are cut into chunks of
// kChunkBytes of input on 32-byte boundaries, which groups of 256 threads take in
// turn: the groups' shares differ by one chunk whatever the tensors' sizes are.
//
// Bound by memory: the input is read for the norm and again, as far as neither
// shared memory nor L2 still has it, to be scaled.  On a B200 (6.56 TB/s for a
// plain copy), as calls among others, floors with one read in brackets:
//   norm of 161 fp32 tensors, 102 MB                   23 us    (15.5)
//   122 MB of fp32 in place, nothing to scale          26 us    (18.6)
//   36 M fp16 into other tensors                       37 us    (22)
//   1 G bf16 into fp32                                 1255 us  (920; 1227 with both reads)
//   1752 fp32 values in seven tensors                  6.4 us, 3.7 on the device: the call
//
// A thread squares the values of one 32-byte load in fp32 and adds the sum to a
// double: a conversion and an addition per load.  Where that sum leaves the
// range in which fp32 keeps all its digits (a value above 2^63, all below
// 2^-30, infinities, NaN) the load's squares are taken again in double, so that
// no norm overflows or vanishes which fp32 can hold.  The partial sums are added
// in a fixed order: the result does not depend on the order of execution.
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>

#include "grad_ops.h"
#include "ibcomm/communicator.h"
#include "kernels.h"
#include "vec_ops.cuh"

namespace ibcomm {
namespace dev {

constexpr int kNormThreads = 256;
// Groups of kNormThreads in a block that sums.  The blocks behind read 296 partial sums instead of 888: where nothing is to
// be scaled (122 MB) they take 5.7 us instead of 7.3.  Clusters of eight that leave one sum do not all fit at once (31 us
// instead of 22 for the sums of 122 MB).
constexpr int kGroups = 3;
constexpr int kBlocksPerSm = 2;  // of those; six of the others
constexpr int kNormCluster = 8;  // blocks of the cluster that takes a short list
constexpr int kChunkBytes = 16384;  // of input: two loads per thread
constexpr double kClipEps = 1e-6;

struct Span {
  const unsigned char* in;  // rounded down to 32 bytes
  unsigned char* out;       // of the same element
  uint64_t begin, end;      // elements from `in` that belong to the tensor
  uint32_t first_chunk;
  uint8_t dtype_in, dtype_out;
  uint8_t vector_out;       // `out` is aligned for vector stores
};

template <int kMost>
struct SpanList {
  uint32_t count;
  uint32_t chunks;
  int in_place;  // every output is its input
  Span span[kMost];
};

// ---- sums ----
// Maxima are kept as the patterns of doubles: of values that are not negative the
// larger one has the larger pattern, and NaN is above them all.  They are whole
// numbers until the end, since arithmetic on a double may give a NaN its sign back.
template <GradPower P> struct Sum { using type = double; };
template <> struct Sum<GradPower::kMax> { using type = long long; };
template <GradPower P> using SumOf = typename Sum<P>::type;

// The pattern of |v|, by words: a mask on the whole is compiled into an absolute
// value, which leaves a NaN's sign.
__device__ __forceinline__ long long Magnitude(double v) {
  return static_cast<long long>((static_cast<unsigned long long>(__double2hiint(v) & 0x7fffffff) << 32) | static_cast<unsigned>(__double2loint(v)));
}

__device__ __forceinline__ double Join(double a, double b) { return a + b; }
__device__ __forceinline__ long long Join(long long a, long long b) { return a > b ? a : b; }

template <GradPower P, typename A, int kN>
__device__ __forceinline__ SumOf<P> JoinValues(SumOf<P> sum, const A* a) {
  if constexpr (P == GradPower::kTwo) {
    if constexpr (sizeof(A) == 4) {
      float s = 0.f, t = 0.f;
#pragma unroll
      for (int e = 0; e < kN; e += 2) {
        s = fmaf(a[e], a[e], s);
        t = fmaf(a[e + 1], a[e + 1], t);
      }
      s += t;
      if (s > 0x1p-60f && s < 0x1p126f) return sum + static_cast<double>(s);
      // Nothing but zeros, as in the rows of an embedding that no token named.
      unsigned any = 0;
#pragma unroll
      for (int e = 0; e < kN; ++e) any |= __float_as_uint(a[e]);
      if ((any & 0x7fffffffu) == 0) return sum;
    }
#pragma unroll
    for (int e = 0; e < kN; ++e) sum = fma(static_cast<double>(a[e]), static_cast<double>(a[e]), sum);
    return sum;
  } else if constexpr (sizeof(A) == 4) {
    unsigned m = 0;
#pragma unroll
    for (int e = 0; e < kN; ++e) m = max(m, __float_as_uint(a[e]) & 0x7fffffffu);
    return Join(sum, Magnitude(static_cast<double>(__uint_as_float(m))));
  } else {
#pragma unroll
    for (int e = 0; e < kN; ++e) sum = Join(sum, Magnitude(a[e]));
    return sum;
  }
}

template <typename S>
__device__ __forceinline__ S WarpJoin(S v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = Join(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}

// The block's sum, in every thread; the order is that of the threads.
template <int kThreads, typename S>
__device__ S BlockJoin(S v, S* shared) {
  v = WarpJoin(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) v = Join(v, shared[w]);
  return v;
}

// ---- chunks ----
template <int kMost>
__device__ __forceinline__ uint32_t SpanOf(const SpanList<kMost>& list, uint32_t chunk) {
  uint32_t lo = 0, hi = list.count;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (list.span[mid].first_chunk <= chunk) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <GradPower P, typename T>
__device__ __forceinline__ SumOf<P> SumChunk(const Span& s, uint32_t chunk, SumOf<P> sum, unsigned char* held) {
  using A = typename Acc<T>::type;
  constexpr int kN = 32 / static_cast<int>(sizeof(T));
  constexpr uint64_t kElems = kChunkBytes / sizeof(T);
  constexpr int kLoads = kChunkBytes / 32 / kNormThreads;
  const uint32_t thread = threadIdx.x % kNormThreads;
  const T* in = reinterpret_cast<const T*>(s.in);
  const uint64_t base = chunk * kElems;
  if (base >= s.begin && base + kElems <= s.end) {
    uint4 lo[kLoads], hi[kLoads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u) Ld32(in + base + (thread + u * kNormThreads) * kN, &lo[u], &hi[u]);
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      A a[kN];
      VecIO<T>::Load(lo[u], a);
      VecIO<T>::Load(hi[u], a + kN / 2);
      sum = JoinValues<P, A, kN>(sum, a);
    }
    if (held != nullptr) {
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        uint4* to = reinterpret_cast<uint4*>(held + (thread + u * kNormThreads) * 32);
        to[0] = lo[u];
        to[1] = hi[u];
      }
    }
    return sum;
  }
#pragma unroll
  for (int u = 0; u < kLoads; ++u) {
    const uint64_t i = base + (thread + u * kNormThreads) * kN;
    A a[kN];
    if (i >= s.begin && i + kN <= s.end) {
      uint4 lo, hi;
      Ld32(in + i, &lo, &hi);
      VecIO<T>::Load(lo, a);
      VecIO<T>::Load(hi, a + kN / 2);
    } else {
#pragma unroll
      for (int e = 0; e < kN; ++e) a[e] = i + e >= s.begin && i + e < s.end ? ToAcc<A, T>(in[i + e]) : A(0);
    }
    sum = JoinValues<P, A, kN>(sum, a);
  }
  return sum;
}

template <typename TI, typename TO>
__device__ __forceinline__ void ScaleChunk(const Span& s, uint32_t chunk, double coefficient, const unsigned char* held) {
  using A = typename Acc<TI>::type;
  using AO = typename Acc<TO>::type;
  constexpr int kWide = static_cast<int>(sizeof(TI) > sizeof(TO) ? sizeof(TI) : sizeof(TO));
  constexpr int kN = 32 / kWide;
  constexpr uint64_t kElems = kChunkBytes / sizeof(TI);
  constexpr int kLoads = static_cast<int>(kElems) / kN / kNormThreads;
  const uint32_t thread = threadIdx.x % kNormThreads;
  const TI* in = reinterpret_cast<const TI*>(s.in);
  TO* out = reinterpret_cast<TO*>(s.out);
  // In fp32 a coefficient below the normal numbers (of gradients near the end of the range) would lose its digits: it is
  // taken 2^126 times as large, and the product is scaled back.
  const bool tiny = sizeof(A) == 4 && coefficient < 0x1p-126;
  const A c = static_cast<A>(tiny ? coefficient * 0x1p126 : coefficient);
  auto scaled = [&](A x) {
    A v = x * c;
    if (tiny) v *= static_cast<A>(0x1p-126);
    return static_cast<AO>(v);
  };
  const uint64_t base = chunk * kElems;
  constexpr bool kWhole = sizeof(TI) * kN == 32;
  struct Raw {
    uint4 v[kWhole ? 2 : 1];
  };
  auto load = [&](uint64_t i, Raw* r) {
    if constexpr (kWhole) Ld32(in + i, &r->v[0], &r->v[1]);
    else r->v[0] = Ld16(in + i);
  };
  auto store = [&](uint64_t i, const Raw& r) {
    A a[kN];
    AO o[kN];
    VecIO<TI>::Load(r.v[0], a);
    if constexpr (kWhole) VecIO<TI>::Load(r.v[1], a + VecIO<TI>::kN);
#pragma unroll
    for (int e = 0; e < kN; ++e) o[e] = scaled(a[e]);
    if constexpr (sizeof(TO) * kN == 32) St32(out + i, VecIO<TO>::Store(o), VecIO<TO>::Store(o + VecIO<TO>::kN));
    else St16(out + i, VecIO<TO>::Store(o));
  };
  if (s.vector_out && base >= s.begin && base + kElems <= s.end) {
    Raw r[kLoads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const uint32_t at = (thread + u * kNormThreads) * kN;
      if (held != nullptr) {
        const uint4* from = reinterpret_cast<const uint4*>(held + at * sizeof(TI));
#pragma unroll
        for (int v = 0; v < (kWhole ? 2 : 1); ++v) r[u].v[v] = from[v];
      } else {
        load(base + at, &r[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < kLoads; ++u) store(base + (thread + u * kNormThreads) * kN, r[u]);
  } else if (s.vector_out) {
    for (int u = 0; u < kLoads; ++u) {
      const uint64_t i = base + (thread + u * kNormThreads) * kN;
      if (i >= s.begin && i + kN <= s.end) {
        Raw r;
        load(i, &r);
        store(i, r);
      } else {
#pragma unroll
        for (int e = 0; e < kN; ++e)
          if (i + e >= s.begin && i + e < s.end) out[i + e] = FromAcc<TO, AO>(scaled(ToAcc<A, TI>(in[i + e])));
      }
    }
  } else {
#pragma unroll 4
    for (uint64_t i = base + thread; i < base + kElems; i += kNormThreads)
      if (i >= s.begin && i < s.end) out[i] = FromAcc<TO, AO>(scaled(ToAcc<A, TI>(in[i])));
  }
}

template <GradPower P, int kMost>
__device__ __forceinline__ SumOf<P> SumRange(const SpanList<kMost>& list, uint32_t first, uint32_t step, unsigned char* held = nullptr, int hold = 0) {
  SumOf<P> sum = 0;
  for (uint32_t c = first; c < list.chunks; c += step, held += kChunkBytes) {
    const Span& s = list.span[SpanOf(list, c)];
    const uint32_t i = c - s.first_chunk;
    unsigned char* here = hold-- > 0 ? held : nullptr;
    switch (static_cast<DType>(s.dtype_in)) {
      case DType::kFloat32: sum = SumChunk<P, float>(s, i, sum, here); break;
      case DType::kFloat64: sum = SumChunk<P, double>(s, i, sum, here); break;
      case DType::kFloat16: sum = SumChunk<P, __half>(s, i, sum, here); break;
      default: sum = SumChunk<P, __nv_bfloat16>(s, i, sum, here); break;
    }
  }
  return sum;
}

template <int kMost>
__device__ __forceinline__ void ScaleAny(const SpanList<kMost>& list, uint32_t chunk, double coefficient, const unsigned char* held = nullptr) {
  const Span& s = list.span[SpanOf(list, chunk)];
  const uint32_t i = chunk - s.first_chunk;
  switch (static_cast<DType>(s.dtype_in)) {
    case DType::kFloat32:
      if (s.dtype_out == static_cast<int>(DType::kFloat32)) ScaleChunk<float, float>(s, i, coefficient, held);
      else if (s.dtype_out == static_cast<int>(DType::kFloat16)) ScaleChunk<float, __half>(s, i, coefficient, held);
      else ScaleChunk<float, __nv_bfloat16>(s, i, coefficient, held);
      break;
    case DType::kFloat64: ScaleChunk<double, double>(s, i, coefficient, held); break;
    case DType::kFloat16:
      if (s.dtype_out == static_cast<int>(DType::kFloat16)) ScaleChunk<__half, __half>(s, i, coefficient, held);
      else ScaleChunk<__half, float>(s, i, coefficient, held);
      break;
    default:
      if (s.dtype_out == static_cast<int>(DType::kBFloat16)) ScaleChunk<__nv_bfloat16, __nv_bfloat16>(s, i, coefficient, held);
      else ScaleChunk<__nv_bfloat16, float>(s, i, coefficient, held);
      break;
  }
}

__device__ __forceinline__ double Coefficient(double norm, double max_norm) {
  const double c = max_norm / (norm + kClipEps);
  return c >= 1.0 ? 1.0 : c;  // a NaN stays
}

struct Finish {
  const double* sums;
  int num_sums;
  void* norm;
  int norm_is_double;
  double* sum;
  double max_norm;
};

// The norm from the sum of everything; one thread of the grid writes the results.
template <GradPower P>
__device__ __forceinline__ double Conclude(const Finish& f, SumOf<P> v) {
  double norm;
  if constexpr (P == GradPower::kTwo) norm = sqrt(v);
  else norm = __longlong_as_double(v);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    if (f.sum != nullptr) *reinterpret_cast<SumOf<P>*>(f.sum) = v;
    if (f.norm != nullptr) {
      if (f.norm_is_double) *static_cast<double*>(f.norm) = norm;
      else *static_cast<float*>(f.norm) = static_cast<float>(norm);
    }
  }
  return norm;
}

// Every warp adds the same partial sums in the same order.
template <GradPower P>
__device__ __forceinline__ double FinishNorm(const Finish& f) {
  const SumOf<P>* sums = reinterpret_cast<const SumOf<P>*>(f.sums);
  SumOf<P> v = 0;
#pragma unroll 4
  for (int i = threadIdx.x & 31; i < f.num_sums; i += 32) v = Join(v, sums[i]);
  return Conclude<P>(f, WarpJoin(v));
}

// partials[block] (+)= the sum of the block's chunks.  The kernel behind is set up while the blocks come to their end.
template <int kMost, GradPower P>
__global__ void __launch_bounds__(kGroups* kNormThreads, kBlocksPerSm)
    GradSumKernel(const __grid_constant__ SpanList<kMost> list, SumOf<P>* partials, int first) {
  __shared__ SumOf<P> shared[kGroups * kNormThreads / 32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const SumOf<P> sum = BlockJoin<kGroups * kNormThreads>(SumRange<P>(list, blockIdx.x * kGroups + threadIdx.x / kNormThreads, gridDim.x * kGroups), shared);
  if (threadIdx.x == 0) partials[blockIdx.x] = first ? sum : Join(partials[blockIdx.x], sum);
}

// The same with the norm at its end, cooperative.  One launch less, which is what
// counts up to 8 MiB (bf16, 2 MiB 8.4 -> 6.7 us, 8 MiB 8.5 -> 8.2); from 16 MiB on
// there is no difference, and from 64 MiB on it is not worth having to wait until
// the whole grid fits beside whatever runs.
template <int kMost, GradPower P>
__global__ void __launch_bounds__(kGroups* kNormThreads, kBlocksPerSm)
    NormKernel(const __grid_constant__ SpanList<kMost> list, SumOf<P>* partials, Finish f) {
  __shared__ SumOf<P> shared[kGroups * kNormThreads / 32];
  const SumOf<P> sum = BlockJoin<kGroups * kNormThreads>(SumRange<P>(list, blockIdx.x * kGroups + threadIdx.x / kNormThreads, gridDim.x * kGroups), shared);
  if (threadIdx.x == 0) partials[blockIdx.x] = sum;
  cooperative_groups::this_grid().sync();
  if (blockIdx.x == 0 && threadIdx.x < 32) FinishNorm<P>(f);
}

template <GradPower P>
__global__ void __launch_bounds__(32) FinishNormKernel(Finish f) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  FinishNorm<P>(f);
}

// Many short blocks: 1 G bf16 into fp32 913 us (6.6 TB/s), with a grid that stays 1020.
template <int kMost, GradPower P>
__global__ void __launch_bounds__(kNormThreads, kGroups* kBlocksPerSm) ClipKernel(const __grid_constant__ SpanList<kMost> list, Finish f, uint32_t per_block) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const double c = Coefficient(FinishNorm<P>(f), f.max_norm);
  // Times one in place: nothing to write.
  if (c == 1.0 && list.in_place) return;
  // From the end: what was read last for the norm is still in L2.
  for (uint32_t u = 0; u < per_block; ++u) {
    const uint32_t i = blockIdx.x * per_block + u;
    if (i < list.chunks) ScaleAny(list, list.chunks - 1 - i, c);
  }
}

// Norm and clipping in one cooperative kernel, a block per SM: the chunks that a
// group of threads reads first stay in shared memory until the norm is known, and
// nothing is launched in between.  Against the two kernels above, on lists of four
// tensors (input, fp32 into other fp32 tensors; nothing to scale):
//   8 MiB   16.2 -> 11.9 us;   9.2 ->  8.6 us
//   64 MiB  35.3 -> 33.1 us;  18.7 -> 17.0 us
//   128 MiB 67.6 -> 63.8 us;  28.8 -> 27.2 us
//   256 MiB    134 -> 132 us; bf16 into fp32 181 -> 184 us
// so lists of up to 128 MiB are taken; above, the shorter blocks of the others win.
constexpr int kHeldGroups = 4, kHeldChunks = 3;  // of a group
constexpr size_t kHeldBytes = static_cast<size_t>(kHeldGroups) * kHeldChunks * kChunkBytes;

template <int kMost, GradPower P>
__global__ void __launch_bounds__(kHeldGroups* kNormThreads, 1)
    HeldClipKernel(const __grid_constant__ SpanList<kMost> list, Finish f, SumOf<P>* partials) {
  extern __shared__ __align__(16) unsigned char memory[];
  __shared__ SumOf<P> shared[kHeldGroups * kNormThreads / 32];
  const uint32_t group = threadIdx.x / kNormThreads, first = blockIdx.x * kHeldGroups + group, step = gridDim.x * kHeldGroups;
  unsigned char* held = memory + group * (kHeldChunks * kChunkBytes);
  const SumOf<P> sum = BlockJoin<kHeldGroups * kNormThreads>(SumRange<P>(list, first, step, held, kHeldChunks), shared);
  if (threadIdx.x == 0) partials[blockIdx.x] = sum;
  cooperative_groups::this_grid().sync();
  const double c = Coefficient(FinishNorm<P>(f), f.max_norm);
  if (c == 1.0 && list.in_place) return;
  // Those that are not held first, from the end: what was read last is still in L2.
  if (first >= list.chunks) return;
  for (uint32_t i = (list.chunks - 1 - first) / step + 1; i-- > 0;) ScaleAny(list, first + i * step, c, i < kHeldChunks ? held + i * kChunkBytes : nullptr);
}

// Few chunks: one cluster does everything, with the blocks' sums in its shared memory.
template <int kMost, GradPower P>
__global__ void __launch_bounds__(kNormThreads) SmallClipKernel(const __grid_constant__ SpanList<kMost> list, Finish f, int clip) {
  __shared__ SumOf<P> shared[kNormThreads / 32], mine;
  const cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
  const SumOf<P> sum = BlockJoin<kNormThreads>(SumRange<P>(list, blockIdx.x, gridDim.x), shared);
  if (threadIdx.x == 0) mine = sum;
  cluster.sync();
  SumOf<P> v = 0;
  for (unsigned b = 0; b < gridDim.x; ++b) v = Join(v, *cluster.map_shared_rank(&mine, b));
  const double norm = Conclude<P>(f, v);
  const double c = Coefficient(norm, f.max_norm);
  if (clip && !(c == 1.0 && list.in_place))
    for (uint32_t i = blockIdx.x; i < list.chunks; i += gridDim.x) ScaleAny(list, i, c);
  cluster.sync();  // nobody reads this block's sum any more
}

}  // namespace dev

namespace {

constexpr uint32_t kSmallChunks = 32;   // that one cluster takes
constexpr uint32_t kMostHeldChunks = 8192;  // 128 MiB
constexpr uint32_t kMostNormChunks = 4096;  // 64 MiB
constexpr uint32_t kMostPerBlock = 8;  // chunks of a block that scales
constexpr int kMostSpans = 800;  // as many fit into the 32764 bytes of a kernel's parameters

uint32_t SizeOf(int dtype) {
  switch (static_cast<DType>(dtype)) {
    case DType::kFloat64: return 8;
    case DType::kFloat32: return 4;
    default: return 2;
  }
}

// Fills `list` from tensors[*next] on; returns whether any is left.
template <int kMost>
void FillList(dev::SpanList<kMost>* list, const GradTensor* tensors, int count, int* next) {
  list->count = 0;
  list->in_place = 1;
  uint64_t chunks = 0;
  for (; *next < count && list->count < kMost; ++*next) {
    const GradTensor& t = tensors[*next];
    if (t.n == 0) continue;
    const uint32_t size = SizeOf(t.dtype_in);
    const uint64_t shift = reinterpret_cast<uintptr_t>(t.in) % 32 / size;
    const uint64_t mine = ((shift + t.n) * size + dev::kChunkBytes - 1) / dev::kChunkBytes;
    if (chunks + mine > 0x7fffffffull) break;
    dev::Span& s = list->span[list->count++];
    s.in = static_cast<const unsigned char*>(t.in) - shift * size;
    s.begin = shift;
    s.end = shift + t.n;
    s.first_chunk = static_cast<uint32_t>(chunks);
    s.dtype_in = static_cast<uint8_t>(t.dtype_in);
    s.dtype_out = static_cast<uint8_t>(t.dtype_out);
    s.out = nullptr;
    s.vector_out = 0;
    if (t.out != t.in || t.dtype_out != t.dtype_in) list->in_place = 0;
    if (t.out != nullptr) {
      const uint32_t size_out = SizeOf(t.dtype_out);
      const uint32_t quantum = 32 / std::max(size, size_out) * size_out;
      // A location before `out` that is only ever used with `begin` added.
      const uintptr_t out = reinterpret_cast<uintptr_t>(t.out) - shift * size_out;
      s.out = reinterpret_cast<unsigned char*>(out);
      s.vector_out = out % quantum == 0;
    }
    chunks += mine;
  }
  list->chunks = static_cast<uint32_t>(chunks);
}

cudaError_t FullGrid(int* blocks) {
  int device = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  *blocks = std::min(sms * dev::kBlocksPerSm, kNormPartials);
  return e;
}

// `early`: the launch is set up while the one before it in the stream comes to its end, and waits before it reads.
template <typename... Params, typename... Args>
cudaError_t Launch(void (*kernel)(Params...), int blocks, int threads, int cluster, bool early, cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(blocks));
  config.blockDim = dim3(static_cast<unsigned>(threads));
  config.stream = stream;
  cudaLaunchAttribute attributes[2];
  config.attrs = attributes;
  if (cluster > 1) {
    cudaLaunchAttribute& a = attributes[config.numAttrs++];
    a.id = cudaLaunchAttributeClusterDimension;
    a.val.clusterDim.x = static_cast<unsigned>(cluster);
    a.val.clusterDim.y = a.val.clusterDim.z = 1;
  }
  if (early) {
    cudaLaunchAttribute& a = attributes[config.numAttrs++];
    a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    a.val.programmaticStreamSerializationAllowed = 1;
  }
  return cudaLaunchKernelEx(&config, kernel, args...);
}

template <int kMost, GradPower P>
cudaError_t LaunchTyped(const GradNormParams& p, cudaStream_t stream) {
  int full = 0;
  cudaError_t e = FullGrid(&full);
  if (e != cudaSuccess) return e;
  dev::SpanList<kMost> list;
  dev::Finish f{p.sums, p.num_sums, p.norm, p.norm_is_double, p.sum, p.max_norm};
  bool first = true;
  if (p.sums == nullptr) {
    f.sums = p.work;
    f.num_sums = full;
    int next = 0;
    do {
      FillList(&list, p.tensors, p.count, &next);
      const bool all = first && next == p.count;
      if (all && list.chunks <= kSmallChunks) {
        const int blocks = static_cast<int>(std::min(std::max(list.chunks, 1u), static_cast<uint32_t>(dev::kNormCluster)));
        return Launch(dev::SmallClipKernel<kMost, P>, blocks, dev::kNormThreads, blocks, false, stream, list, f, p.clip ? 1 : 0);
      }
      if (all && p.clip && list.chunks <= kMostHeldChunks) {
        f.num_sums = full / dev::kBlocksPerSm;
        e = AllowSharedMemory(dev::HeldClipKernel<kMost, P>, dev::kHeldBytes);
        if (e != cudaSuccess) return e;
        e = LaunchTogether(dev::HeldClipKernel<kMost, P>, f.num_sums, dev::kHeldGroups * dev::kNormThreads, dev::kHeldBytes, stream, list, f,
                           reinterpret_cast<dev::SumOf<P>*>(p.work));
        if (e != cudaErrorCooperativeLaunchTooLarge) return e;
      }
      if (all) f.num_sums = static_cast<int>(std::min<uint64_t>(full, (list.chunks + dev::kGroups - 1) / dev::kGroups));
      if (all && !p.clip && list.chunks <= kMostNormChunks) {
        e = LaunchTogether(dev::NormKernel<kMost, P>, f.num_sums, dev::kGroups * dev::kNormThreads, 0, stream, list, reinterpret_cast<dev::SumOf<P>*>(p.work), f);
        if (e != cudaErrorCooperativeLaunchTooLarge) return e;
      }
      // The first launch of a call is an ordinary one: what it reads is written by whatever came before.
      e = Launch(dev::GradSumKernel<kMost, P>, f.num_sums, dev::kGroups * dev::kNormThreads, 1, !first, stream, list, reinterpret_cast<dev::SumOf<P>*>(p.work),
                 first ? 1 : 0);
      if (e != cudaSuccess) return e;
      first = false;
    } while (next < p.count);
  }
  if (!p.clip) return Launch(dev::FinishNormKernel<P>, 1, 32, 1, !first, stream, f);
  int next = 0;
  do {
    FillList(&list, p.tensors, p.count, &next);
    const uint32_t per_block = std::min(std::max(list.chunks / static_cast<uint32_t>(2 * dev::kGroups * full), 1u), kMostPerBlock);
    const int blocks = static_cast<int>(std::max((list.chunks + per_block - 1) / per_block, 1u));
    // Behind the sums of the same call, or on its own.
    e = Launch(dev::ClipKernel<kMost, P>, blocks, dev::kNormThreads, 1, !first, stream, list, f, per_block);
    if (e != cudaSuccess) return e;
    first = true;
  } while (next < p.count);
  return cudaSuccess;
}

template <int kMost>
cudaError_t LaunchSized(const GradNormParams& p, cudaStream_t stream) {
  return p.power == GradPower::kTwo ? LaunchTyped<kMost, GradPower::kTwo>(p, stream) : LaunchTyped<kMost, GradPower::kMax>(p, stream);
}

}  // namespace

cudaError_t LaunchGradNorm(const GradNormParams& p, cudaStream_t stream) {
  // A short list has a short block of parameters.
  if (p.count <= 16) return LaunchSized<16>(p, stream);
  return p.count <= 64 ? LaunchSized<64>(p, stream) : p.count <= 256 ? LaunchSized<256>(p, stream) : LaunchSized<kMostSpans>(p, stream);
}

}  // namespace ibcomm
