// The norm of a list of tensors taken as one vector, and clipping:
//   N = sqrt(sum x^2)  (or max |x|),   out = round(x * min(1, max_norm / (N + 1e-6))).
//
// The list travels in the kernel's parameters (nothing is copied ahead of the
// launch, and a captured call keeps its own).  Tensors are cut into chunks of
// kChunkBytes of input on 32-byte boundaries; a block works on a contiguous
// range of chunks, so the ranges differ by one chunk at most whatever the
// tensors' sizes are.
//
// A thread squares the values of one 32-byte load in fp32 and adds the sum to a
// double: a conversion and an addition per load.  Where that sum leaves the
// range in which fp32 keeps all its digits (a value above 2^63, all below
// 2^-30, infinities, NaN) the load's squares are taken again in double, so that
// no norm overflows or vanishes which fp32 can hold.  The partial sums are added
// in a fixed order: the result does not depend on the order of execution.
#include <algorithm>
#include <cmath>

#include "grad_ops.h"
#include "ibcomm/communicator.h"
#include "vec_ops.cuh"

namespace ibcomm {
namespace dev {

constexpr int kNormThreads = 256;
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

// The block's sum, in every thread; the order is that of the threads.
template <typename S>
__device__ S BlockJoin(S v, S* shared) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = Join(v, __shfl_xor_sync(0xffffffffu, v, d));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < kNormThreads / 32; ++w) v = Join(v, shared[w]);
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
__device__ __forceinline__ SumOf<P> SumChunk(const Span& s, uint32_t chunk, SumOf<P> sum) {
  using A = typename Acc<T>::type;
  constexpr int kN = 32 / static_cast<int>(sizeof(T));
  constexpr uint64_t kElems = kChunkBytes / sizeof(T);
  constexpr int kLoads = kChunkBytes / 32 / kNormThreads;
  const T* in = reinterpret_cast<const T*>(s.in);
  const uint64_t base = chunk * kElems;
  if (base >= s.begin && base + kElems <= s.end) {
    uint4 lo[kLoads], hi[kLoads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u) Ld32(in + base + (threadIdx.x + u * kNormThreads) * kN, &lo[u], &hi[u]);
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      A a[kN];
      VecIO<T>::Load(lo[u], a);
      VecIO<T>::Load(hi[u], a + kN / 2);
      sum = JoinValues<P, A, kN>(sum, a);
    }
    return sum;
  }
#pragma unroll
  for (int u = 0; u < kLoads; ++u) {
    const uint64_t i = base + (threadIdx.x + u * kNormThreads) * kN;
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
__device__ __forceinline__ void ScaleChunk(const Span& s, uint32_t chunk, double coefficient) {
  using A = typename Acc<TI>::type;
  using AO = typename Acc<TO>::type;
  constexpr int kWide = static_cast<int>(sizeof(TI) > sizeof(TO) ? sizeof(TI) : sizeof(TO));
  constexpr int kN = 32 / kWide;
  constexpr uint64_t kElems = kChunkBytes / sizeof(TI);
  constexpr int kLoads = static_cast<int>(kElems) / kN / kNormThreads;
  const TI* in = reinterpret_cast<const TI*>(s.in);
  TO* out = reinterpret_cast<TO*>(s.out);
  const A c = static_cast<A>(coefficient);
  const uint64_t base = chunk * kElems;
  if (s.vector_out) {
#pragma unroll 2
    for (int u = 0; u < kLoads; ++u) {
      const uint64_t i = base + (threadIdx.x + u * kNormThreads) * kN;
      if (i >= s.begin && i + kN <= s.end) {
        A a[kN];
        AO o[kN];
        if constexpr (sizeof(TI) * kN == 32) {
          uint4 lo, hi;
          Ld32(in + i, &lo, &hi);
          VecIO<TI>::Load(lo, a);
          VecIO<TI>::Load(hi, a + VecIO<TI>::kN);
        } else {
          VecIO<TI>::Load(Ld16(in + i), a);
        }
#pragma unroll
        for (int e = 0; e < kN; ++e) o[e] = static_cast<AO>(a[e] * c);
        if constexpr (sizeof(TO) * kN == 32) St32(out + i, VecIO<TO>::Store(o), VecIO<TO>::Store(o + VecIO<TO>::kN));
        else St16(out + i, VecIO<TO>::Store(o));
      } else {
#pragma unroll
        for (int e = 0; e < kN; ++e)
          if (i + e >= s.begin && i + e < s.end) out[i + e] = FromAcc<TO, AO>(static_cast<AO>(ToAcc<A, TI>(in[i + e]) * c));
      }
    }
  } else {
#pragma unroll 4
    for (uint64_t i = base + threadIdx.x; i < base + kElems; i += kNormThreads)
      if (i >= s.begin && i < s.end) out[i] = FromAcc<TO, AO>(static_cast<AO>(ToAcc<A, TI>(in[i]) * c));
  }
}

// The block's chunks: a contiguous range.
__device__ __forceinline__ uint32_t RangeBegin(uint32_t chunks, uint32_t block) {
  return static_cast<uint32_t>(static_cast<uint64_t>(chunks) * block / gridDim.x);
}

// partials[block] (+)= the sum of the block's chunks.
template <int kMost, GradPower P>
__global__ void __launch_bounds__(kNormThreads) GradSumKernel(const __grid_constant__ SpanList<kMost> list, SumOf<P>* partials, int first) {
  __shared__ SumOf<P> shared[kNormThreads / 32];
  uint32_t c = RangeBegin(list.chunks, blockIdx.x);
  const uint32_t end = RangeBegin(list.chunks, blockIdx.x + 1);
  SumOf<P> sum = 0;
  uint32_t k = c < end ? SpanOf(list, c) : 0;
  for (; c < end; ++c) {
    while (k + 1 < list.count && list.span[k + 1].first_chunk <= c) ++k;
    const Span& s = list.span[k];
    const uint32_t i = c - s.first_chunk;
    switch (static_cast<DType>(s.dtype_in)) {
      case DType::kFloat32: sum = SumChunk<P, float>(s, i, sum); break;
      case DType::kFloat64: sum = SumChunk<P, double>(s, i, sum); break;
      case DType::kFloat16: sum = SumChunk<P, __half>(s, i, sum); break;
      default: sum = SumChunk<P, __nv_bfloat16>(s, i, sum); break;
    }
  }
  sum = BlockJoin(sum, shared);
  if (threadIdx.x == 0) partials[blockIdx.x] = first ? sum : Join(partials[blockIdx.x], sum);
}

struct Finish {
  const double* sums;
  int num_sums;
  void* norm;
  int norm_is_double;
  double* sum;
  double max_norm;
};

// The sum of all partial sums, in every thread of every block; block 0 writes the results.
template <GradPower P>
__device__ __forceinline__ double FinishNorm(const Finish& f, SumOf<P>* shared) {
  const SumOf<P>* sums = reinterpret_cast<const SumOf<P>*>(f.sums);
  SumOf<P> v = 0;
  for (int i = threadIdx.x; i < f.num_sums; i += kNormThreads) v = Join(v, sums[i]);
  v = BlockJoin(v, shared);
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

template <GradPower P>
__global__ void __launch_bounds__(kNormThreads) FinishNormKernel(Finish f) {
  __shared__ SumOf<P> shared[kNormThreads / 32];
  FinishNorm<P>(f, shared);
}

template <int kMost, GradPower P>
__global__ void __launch_bounds__(kNormThreads) ClipKernel(const __grid_constant__ SpanList<kMost> list, Finish f) {
  __shared__ SumOf<P> shared[kNormThreads / 32];
  const double norm = FinishNorm<P>(f, shared);
  double coefficient = f.max_norm / (norm + kClipEps);
  if (coefficient >= 1.0) coefficient = 1.0;  // a NaN stays
  // From the range's end: what was read last for the norm is still in L2.
  const uint32_t begin = RangeBegin(list.chunks, blockIdx.x);
  uint32_t c = RangeBegin(list.chunks, blockIdx.x + 1);
  uint32_t k = c > begin ? SpanOf(list, c - 1) : 0;
  while (c > begin) {
    --c;
    while (list.span[k].first_chunk > c) --k;
    const Span& s = list.span[k];
    const uint32_t i = c - s.first_chunk;
    // Times one in place: nothing to write.
    if (coefficient == 1.0 && s.in == s.out && s.dtype_in == s.dtype_out) continue;
    switch (static_cast<DType>(s.dtype_in)) {
      case DType::kFloat32:
        if (s.dtype_out == static_cast<int>(DType::kFloat32)) ScaleChunk<float, float>(s, i, coefficient);
        else if (s.dtype_out == static_cast<int>(DType::kFloat16)) ScaleChunk<float, __half>(s, i, coefficient);
        else ScaleChunk<float, __nv_bfloat16>(s, i, coefficient);
        break;
      case DType::kFloat64: ScaleChunk<double, double>(s, i, coefficient); break;
      case DType::kFloat16:
        if (s.dtype_out == static_cast<int>(DType::kFloat16)) ScaleChunk<__half, __half>(s, i, coefficient);
        else ScaleChunk<__half, float>(s, i, coefficient);
        break;
      default:
        if (s.dtype_out == static_cast<int>(DType::kBFloat16)) ScaleChunk<__nv_bfloat16, __nv_bfloat16>(s, i, coefficient);
        else ScaleChunk<__nv_bfloat16, float>(s, i, coefficient);
        break;
    }
  }
}

}  // namespace dev

namespace {

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
  uint64_t chunks = 0;
  for (; *next < count && list->count < kMost; ++*next) {
    const GradTensor& t = tensors[*next];
    if (t.n == 0) continue;
    const uint32_t size = SizeOf(t.dtype_in);
    const uint64_t shift = reinterpret_cast<uintptr_t>(t.in) % 32 / size;
    const uint64_t mine = ((shift + t.n) * size + dev::kChunkBytes - 1) / dev::kChunkBytes;
    if (chunks + mine > 0xffffffffull) break;
    dev::Span& s = list->span[list->count++];
    s.in = static_cast<const unsigned char*>(t.in) - shift * size;
    s.begin = shift;
    s.end = shift + t.n;
    s.first_chunk = static_cast<uint32_t>(chunks);
    s.dtype_in = static_cast<uint8_t>(t.dtype_in);
    s.dtype_out = static_cast<uint8_t>(t.dtype_out);
    s.out = nullptr;
    s.vector_out = 0;
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
  *blocks = std::min(sms * 8, kNormPartials);
  return e;
}

template <int kMost, GradPower P>
cudaError_t LaunchTyped(const GradNormParams& p, cudaStream_t stream) {
  int full = 0;
  cudaError_t e = FullGrid(&full);
  if (e != cudaSuccess) return e;
  dev::SpanList<kMost> list;
  dev::Finish f{p.sums, p.num_sums, p.norm, p.norm_is_double, p.sum, p.max_norm};
  if (p.sums == nullptr) {
    f.sums = p.work;
    f.num_sums = full;
    int next = 0;
    bool first = true;
    do {
      FillList(&list, p.tensors, p.count, &next);
      int blocks = full;
      if (first && next == p.count) blocks = f.num_sums = static_cast<int>(std::min<uint64_t>(full, std::max<uint32_t>(list.chunks, 1)));
      dev::GradSumKernel<kMost, P><<<blocks, dev::kNormThreads, 0, stream>>>(list, reinterpret_cast<dev::SumOf<P>*>(p.work), first ? 1 : 0);
      if ((e = cudaGetLastError()) != cudaSuccess) return e;
      first = false;
    } while (next < p.count);
  }
  if (!p.clip) {
    dev::FinishNormKernel<P><<<1, dev::kNormThreads, 0, stream>>>(f);
    return cudaGetLastError();
  }
  int next = 0;
  do {
    FillList(&list, p.tensors, p.count, &next);
    const int blocks = static_cast<int>(std::min<uint64_t>(full, std::max<uint32_t>(list.chunks, 1)));
    dev::ClipKernel<kMost, P><<<blocks, dev::kNormThreads, 0, stream>>>(list, f);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
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
  return p.count <= 16 ? LaunchSized<16>(p, stream) : LaunchSized<kMostSpans>(p, stream);
}

}  // namespace ibcomm
