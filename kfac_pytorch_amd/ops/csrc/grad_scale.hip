// One norm, or one inner product, over many tensors, and the rescale by it.
//
//   clip:        norm = (sum_i |a_i|^p)^(1/p),  out = a min(1, max/(norm+1e-6))
//   trust region: nu = min(1, sqrt(kl / |lr^2 sum_i u_i g_i|)),  out = u nu
//
// Two passes over the data and a step of one block between them; nothing
// waits for the host.  A pass is a few launches whatever the number of
// tensors: their addresses and shapes travel in the kernel's arguments, and a
// workgroup finds its tensor by bisection.  Tensors that follow each other in
// memory (views of a bucket) are merged on the host first.
//
// Sums are in double: squares of fp32 neither overflow nor vanish, and the
// result does not depend on how the tensors were cut up beyond its last bits.
// Each workgroup leaves one sum; they are added in a fixed order, so the same
// call gives the same bits.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <hip/hip_runtime.h>

#include <ATen/MemoryOverlap.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <optional>
#include <tuple>
#include <vector>

namespace {

using torch::Tensor;

void check_hip(hipError_t e) {
  TORCH_CHECK(e == hipSuccess, "HIP error: ", hipGetErrorString(e));
}

constexpr int THREADS = 256;
// 16-byte groups a lane has in flight; 8 leave too few workgroups to a CU (the
// inner product of 25 M pairs: 36 us with 4, 48 with 8)
constexpr int UNROLL = 4;
constexpr int CHUNK = THREADS * UNROLL;    // groups of a chunk
constexpr int MOST_BLOCKS = 8192;

// NP operands seen as rows x columns, neighbouring columns next to each other,
// in groups of 16 bytes of the first operand.
template <int NP>
struct Entry {
  const void* p[NP];
  int ld[NP];             // values from a row to the next
  unsigned rows, groups;  // groups of a row
  unsigned tail;          // values of a row's last group
  unsigned start;         // first chunk
};

// kernel arguments stay below 4 KB
template <int NP>
struct List {
  static constexpr int MAX = (4096 - 128) / sizeof(Entry<NP>);
  int n;
  unsigned chunks, per;   // chunks in all, and for each block
  Entry<NP> e[MAX];
};

template <class T, int N>
struct Pack {
  T v[N];
};

// `have` values from p on, the rest zeros; any alignment
template <class T, int N>
__device__ __forceinline__ void fetch(const T* p, int have, float (&f)[N]) {
  Pack<T, N> t;
  if (have == N) {
    __builtin_memcpy(&t, p, sizeof(t));
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = (float)t.v[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = i < have ? (float)p[i] : 0.f;
  }
}

template <class T, int N>
__device__ __forceinline__ void put(T* p, int have, const float (&f)[N]) {
  Pack<T, N> t;
#pragma unroll
  for (int i = 0; i < N; ++i) t.v[i] = (T)f[i];
  if (have == N) {
    // past the caches: what is written is not read again soon, what the
    // second pass reads is there (54 M values: 69 us against 76)
    using W = __attribute__((ext_vector_type(4), aligned(alignof(T)))) int;
    if constexpr (sizeof(t) == 16) {
      __builtin_nontemporal_store(__builtin_bit_cast(W, t), (W*)p);
    } else {
      __builtin_memcpy(p, &t, sizeof(t));
    }
  } else {
    for (int i = 0; i < have; ++i) p[i] = t.v[i];
  }
}

template <int NP>
__device__ __forceinline__ int find(const List<NP>& list, unsigned chunk) {
  int lo = 0, hi = list.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (list.e[mid].start <= chunk) {
      lo = mid;
    } else {
      hi = mid - 1;
    }
  }
  return lo;
}

struct Place {
  unsigned row;
  unsigned long col;
  int have;  // values of the group, 0 past the end
};

template <int NP, int N>
__device__ __forceinline__ Place place(const Entry<NP>& e, unsigned chunk,
                                       int k) {
  const unsigned long g = (unsigned long)(chunk - e.start) * CHUNK +
                          (unsigned)(k * THREADS) + threadIdx.x;
  Place at;
  unsigned in;  // group within its row
  bool there;
  if (e.rows == 1) {
    at.row = 0;
    in = (unsigned)g;
    there = g < e.groups;
  } else {
    // the host keeps rows * groups below 2^32
    at.row = (unsigned)g / e.groups;
    in = (unsigned)g - at.row * e.groups;
    there = g < (unsigned long)e.rows * e.groups;
  }
  at.col = (unsigned long)in * N;
  at.have = !there ? 0 : in == e.groups - 1 ? (int)e.tail : N;
  return at;
}

enum Kind { SQUARES, ABSOLUTES, LARGEST };

// a maximum that keeps a NaN
__device__ __forceinline__ double larger(double a, double b) {
  return (a > b || a != a) ? a : b;
}

template <int KIND>
__device__ __forceinline__ double block_reduce(double s) {
  __shared__ double part[16];
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) {
    const double o = __shfl_xor(s, k);
    s = KIND == LARGEST ? larger(s, o) : s + o;
  }
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  double t = part[0];
  for (unsigned k = 1; k < blockDim.x >> 6; ++k) {
    t = KIND == LARGEST ? larger(t, part[k]) : t + part[k];
  }
  return t;
}

template <class T, int KIND>
__global__ __launch_bounds__(THREADS) void norm_kernel(
    const List<1> list, double* __restrict__ sums) {
  constexpr int N = 16 / sizeof(T);
  double s = 0.0;
  for (unsigned j = 0; j < list.per; ++j) {
    const unsigned chunk = blockIdx.x * list.per + j;
    if (chunk >= list.chunks) break;
    const Entry<1>& e = list.e[find(list, chunk)];
    float f[UNROLL][N];
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      const Place at = place<1, N>(e, chunk, k);
      fetch((const T*)e.p[0] + (long)at.row * e.ld[0] + at.col, at.have, f[k]);
    }
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const double v = (double)f[k][i];
        if constexpr (KIND == SQUARES) {
          s = fma(v, v, s);
        } else if constexpr (KIND == ABSOLUTES) {
          s += fabs(v);
        } else {
          s = larger(s, fabs(v));
        }
      }
    }
  }
  s = block_reduce<KIND>(s);
  if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

template <class U, class G>
__global__ __launch_bounds__(THREADS) void dot_kernel(
    const List<2> list, double* __restrict__ sums) {
  constexpr int N = 16 / sizeof(U);
  double s = 0.0;
  for (unsigned j = 0; j < list.per; ++j) {
    const unsigned chunk = blockIdx.x * list.per + j;
    if (chunk >= list.chunks) break;
    const Entry<2>& e = list.e[find(list, chunk)];
    float u[UNROLL][N], g[UNROLL][N];
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      const Place at = place<2, N>(e, chunk, k);
      fetch((const U*)e.p[0] + (long)at.row * e.ld[0] + at.col, at.have, u[k]);
      fetch((const G*)e.p[1] + (long)at.row * e.ld[1] + at.col, at.have, g[k]);
    }
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        s = fma((double)u[k][i], (double)g[k][i], s);
      }
    }
  }
  s = block_reduce<SQUARES>(s);
  if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

// one block: result[0] = norm, result[1] = factor
template <int KIND>
__global__ __launch_bounds__(1024) void norm_end_kernel(
    const double* __restrict__ sums, int n, double max_norm,
    float* __restrict__ result) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += 1024) {
    s = KIND == LARGEST ? larger(s, sums[i]) : s + sums[i];
  }
  s = block_reduce<KIND>(s);
  if (threadIdx.x == 0) {
    const double norm = KIND == SQUARES ? sqrt(s) : s;
    const double f = max_norm / (norm + 1e-6);
    result[0] = (float)norm;
    result[1] = (float)(f > 1.0 ? 1.0 : f);  // NaN stays
  }
}

// one block: result[0] = result[1] = nu
__global__ __launch_bounds__(1024) void trust_end_kernel(
    const double* __restrict__ sums, int n, double lr, double kl,
    float* __restrict__ result) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += 1024) s += sums[i];
  s = block_reduce<SQUARES>(s);
  if (threadIdx.x == 0) {
    double a = fabs(s * lr * lr);
    a = a < 1e-30 ? 1e-30 : a;               // NaN stays
    const double r = sqrt(kl / a);
    result[0] = result[1] = (float)(r > 1.0 ? 1.0 : r);
  }
}

// out = in * result[1].  The chunks are taken last first: the end of what the
// first pass read is what the card's last cache still holds.
template <class I, class O>
__global__ __launch_bounds__(THREADS) void scale_kernel(
    const List<2> list, const float* __restrict__ result) {
  constexpr int N = 16 / sizeof(I);
  const float f = result[1];
  for (unsigned j = 0; j < list.per; ++j) {
    const unsigned id = blockIdx.x * list.per + j;
    if (id >= list.chunks) break;
    const unsigned chunk = list.chunks - 1 - id;
    const Entry<2>& e = list.e[find(list, chunk)];
    if (f == 1.f && sizeof(I) == sizeof(O) && e.p[0] == e.p[1] &&
        e.ld[0] == e.ld[1]) {
      continue;  // in place, nothing to do
    }
    float v[UNROLL][N];
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      const Place at = place<2, N>(e, chunk, k);
      fetch((const I*)e.p[0] + (long)at.row * e.ld[0] + at.col, at.have, v[k]);
    }
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      const Place at = place<2, N>(e, chunk, k);
#pragma unroll
      for (int i = 0; i < N; ++i) v[k][i] *= f;
      put((O*)const_cast<void*>(e.p[1]) + (long)at.row * e.ld[1] + at.col, at.have,
          v[k]);
    }
  }
}

// ------------------------------------------------------------------- host
template <int NP>
struct Item {
  Entry<NP> e;
  long cols;
};

// Several operands of one shape as rows x cols with unit column stride; false
// where they are not so, and the caller copies them: a few launches a tensor
// (ResNet-50's updates and channels-last gradients: 301 us; of one order: 90).
template <int NP>
bool as_rows(const std::array<const Tensor*, NP>& t, Item<NP>* item) {
  Entry<NP>* e = &item->e;
  bool dense = true;
  for (int i = 0; i < NP; ++i) dense &= t[i]->is_contiguous();
  if (dense) {
    item->cols = t[0]->numel();
    e->rows = 1;
    for (int i = 0; i < NP; ++i) {
      e->p[i] = t[i]->const_data_ptr();
      e->ld[i] = 0;
    }
    return true;
  }
  const auto sizes = t[0]->sizes();
  // dims of more than one value, largest stride of the first operand first
  std::vector<int> dims;
  for (int d = 0; d < (int)sizes.size(); ++d) {
    if (sizes[d] != 1) dims.push_back(d);
  }
  std::stable_sort(dims.begin(), dims.end(), [&](int a, int b) {
    return t[NP - 1]->stride(a) > t[NP - 1]->stride(b);
  });
  // merge neighbours that every operand lays one after the other
  struct Dim {
    long size;
    long stride[NP];
  };
  std::vector<Dim> kept;
  for (int d : dims) {
    Dim now{sizes[d], {}};
    for (int i = 0; i < NP; ++i) now.stride[i] = t[i]->stride(d);
    if (!kept.empty()) {
      bool joins = true;
      for (int i = 0; i < NP; ++i) {
        joins &= kept.back().stride[i] == now.stride[i] * now.size;
      }
      if (joins) {
        now.size *= kept.back().size;
        kept.pop_back();
      }
    }
    kept.push_back(now);
  }
  bool unit = !kept.empty();
  for (int i = 0; i < NP && unit; ++i) unit = kept.back().stride[i] == 1;
  if (!unit) {  // a column of one value
    kept.push_back(Dim{1, {}});
    for (int i = 0; i < NP; ++i) kept.back().stride[i] = 1;
  }
  if (kept.size() > 2) return false;
  const long rows = kept.size() == 2 ? kept[0].size : 1;
  item->cols = kept.back().size;
  for (int i = 0; i < NP; ++i) {
    e->p[i] = t[i]->const_data_ptr();
    const long ld = kept.size() == 2 ? kept[0].stride[i] : 0;
    if (ld >= (1l << 31)) return false;
    e->ld[i] = (int)ld;
  }
  if (rows >= (1l << 31)) return false;
  e->rows = (unsigned)rows;
  return true;
}

template <int NP>
struct Batch {
  std::vector<Item<NP>> items;

  // sizes: bytes of a value of each operand
  void add(const Item<NP>& item, const std::array<long, NP>& sizes) {
    if (!items.empty() && item.e.rows == 1 && items.back().e.rows == 1 &&
        items.back().cols + item.cols < (1l << 33)) {
      Item<NP>& last = items.back();
      bool joins = true;
      for (int i = 0; i < NP; ++i) {
        joins &= (const char*)last.e.p[i] + last.cols * sizes[i] ==
                 (const char*)item.e.p[i];
      }
      if (joins) {
        last.cols += item.cols;
        return;
      }
    }
    items.push_back(item);
  }

  // groups of `n` values
  void group(int n) {
    for (auto& item : items) {
      const long g = (item.cols + n - 1) / n;
      TORCH_CHECK(g < (1l << 32) &&
                      (item.e.rows == 1 || g * item.e.rows < (1l << 32)),
                  "tensor too large");
      item.e.groups = (unsigned)g;
      item.e.tail = (unsigned)(item.cols - (g - 1) * n);
    }
  }

  template <class F>
  void launch(F f) {
    for (size_t first = 0; first < items.size();
         first += List<NP>::MAX) {
      List<NP> list;
      list.n = (int)std::min<size_t>(List<NP>::MAX, items.size() - first);
      unsigned at = 0;
      for (int i = 0; i < list.n; ++i) {
        list.e[i] = items[first + i].e;
        list.e[i].start = at;
        at += (unsigned)(((unsigned long)list.e[i].rows *
                              list.e[i].groups + CHUNK - 1) / CHUNK);
      }
      list.chunks = at;
      list.per = (at + MOST_BLOCKS - 1) / MOST_BLOCKS;
      f(list, (int)((at + list.per - 1) / list.per));
    }
  }

  int blocks() {
    int n = 0;
    launch([&](const List<NP>&, int b) { n += b; });
    return n;
  }
};

template <class F>
void by_type(at::ScalarType t, F f) {
  switch (t) {
    case at::kFloat: f((float*)nullptr); break;
    case at::kBFloat16: f((__bf16*)nullptr); break;
    case at::kHalf: f((_Float16*)nullptr); break;
    default: TORCH_CHECK(false, "unsupported dtype ", t);
  }
}

// Lists of dense tensors on one GPU, pairwise of one shape; those to be
// written have no two values at one place, and none is there twice.
void check_lists(const char* name,
                 std::initializer_list<const std::vector<Tensor>*> lists) {
  const std::vector<Tensor>& first = **lists.begin();
  for (const auto* list : lists) {
    TORCH_CHECK_VALUE(list->size() == first.size(), name, ": lists of ",
                      first.size(), " and ", list->size(), " tensors");
    for (size_t i = 0; i < first.size(); ++i) {
      const Tensor& t = (*list)[i];
      TORCH_CHECK_VALUE(t.device() == first[0].device(), name,
                        ": tensors on ", first[0].device(), " and ",
                        t.device());
      const auto type = t.scalar_type();
      TORCH_CHECK_TYPE(t.layout() == at::kStrided &&
                           (type == at::kFloat || type == at::kBFloat16 ||
                            type == at::kHalf),
                       name, ": dense fp32, bf16 or fp16 expected on the "
                             "GPU, got ", type, ", ", t.layout());
      TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), name,
                                  " has no forward-mode derivative");
      TORCH_CHECK_VALUE(list == &first || t.sizes() == first[i].sizes(),
                        name, ": shapes ", first[i].sizes(), " and ",
                        t.sizes(), " differ");
      // sharded or fake tensors name a device and have no memory there
      TORCH_CHECK_TYPE(t.numel() == 0 || t.const_data_ptr() != nullptr, name,
                       ": tensors with memory of their own expected");
    }
  }
}

// What is written: no place twice, and none of an input but its own, as it
// lies (in place).  Of tensors with gaps, which may be woven into each other,
// only the first value is looked at.
void check_outputs(const char* name, const std::vector<Tensor>& in,
                   const std::vector<Tensor>& out) {
  struct Range {
    const char *begin, *end;
  };
  const auto range = [](const Tensor& t) {
    const char* begin = (const char*)t.const_data_ptr();
    const bool dense = t.is_contiguous() || t.is_non_overlapping_and_dense();
    return Range{begin, begin + (dense ? t.numel() : 1) * t.element_size()};
  };
  std::vector<Range> written;
  written.reserve(out.size());
  for (const Tensor& t : out) {
    TORCH_CHECK_VALUE(t.is_contiguous() || at::has_internal_overlap(t) !=
                                               at::MemOverlap::Yes,
                      name, ": an output's values share memory");
    if (t.numel()) written.push_back(range(t));
  }
  std::sort(written.begin(), written.end(),
            [](const Range& a, const Range& b) { return a.begin < b.begin; });
  for (size_t i = 1; i < written.size(); ++i) {
    TORCH_CHECK_VALUE(written[i].begin >= written[i - 1].end, name,
                      ": the same memory is to be written twice");
  }
  for (size_t i = 0; i < in.size(); ++i) {
    if (in[i].numel() == 0 ||
        (in[i].const_data_ptr() == out[i].const_data_ptr() &&
         in[i].scalar_type() == out[i].scalar_type() &&
         in[i].strides() == out[i].strides())) {
      continue;
    }
    const Range r = range(in[i]);
    const auto after = std::lower_bound(
        written.begin(), written.end(), r.end,
        [](const Range& w, const char* end) { return w.begin < end; });
    TORCH_CHECK_VALUE(after == written.begin() || (after - 1)->end <= r.begin,
                      name, ": an output shares memory with another input");
  }
}

constexpr at::ScalarType TYPES[] = {at::kFloat, at::kBFloat16, at::kHalf};

// The imaginary part of a lazy conjugate is memory with a sign pending on it.
// The kernels read and write memory, which is right where both operands have
// the sign or neither has.
bool other_sign(const Tensor& a, const Tensor& b) {
  return a.is_neg() != b.is_neg();
}

template <int NP>
Item<NP> must(const std::array<const Tensor*, NP>& t) {
  Item<NP> e{};
  TORCH_CHECK(as_rows<NP>(t, &e), "tensor layout");
  return e;
}

void scale_pass(const std::vector<Tensor>& in, const std::vector<Tensor>& out,
                const float* result, hipStream_t s) {
  std::vector<std::pair<Tensor, Tensor>> copies;
  for (at::ScalarType ti : TYPES) {
    for (at::ScalarType to : TYPES) {
      Batch<2> batch;
      for (size_t i = 0; i < in.size(); ++i) {
        if (in[i].scalar_type() != ti || out[i].scalar_type() != to ||
            in[i].numel() == 0) {
          continue;
        }
        Item<2> e{};
        if (other_sign(in[i], out[i]) || !as_rows<2>({&in[i], &out[i]}, &e)) {
          Tensor a = in[i].resolve_neg().contiguous();
          Tensor b = at::empty(out[i].sizes(), out[i].options());
          e = must<2>({&a, &b});
          copies.emplace_back(out[i], b);
          copies.emplace_back(Tensor(), a);  // kept until the launches
        }
        batch.add(e, {(long)in[i].element_size(),
                      (long)out[i].element_size()});
      }
      if (batch.items.empty()) continue;
      by_type(ti, [&](auto* pi) {
        using I = std::remove_pointer_t<decltype(pi)>;
        by_type(to, [&](auto* po) {
          using O = std::remove_pointer_t<decltype(po)>;
          batch.group(16 / sizeof(I));
          batch.launch([&](const List<2>& list, int blocks) {
            scale_kernel<I, O><<<blocks, THREADS, 0, s>>>(list, result);
            check_hip(hipGetLastError());
          });
        });
      });
    }
  }
  for (auto& c : copies) {
    if (c.first.defined()) c.first.copy_(c.second);
  }
  // autograd sees that these were written
  for (const Tensor& t : out) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  }
}

}  // namespace

// -> [norm, factor]; writes out where given
Tensor grad_norm(std::vector<Tensor> tensors,
                 std::optional<std::vector<Tensor>> out, double max_norm,
                 int64_t kind) {
  TORCH_CHECK_VALUE(!tensors.empty(), "grad_norm: no tensors");
  if (out) {
    check_lists("clip_by_global_norm", {&tensors, &*out});
    check_outputs("clip_by_global_norm", tensors, *out);
  } else {
    check_lists("global_norm", {&tensors});
  }
  const c10::OptionalDeviceGuard guard(tensors[0].device());
  const hipStream_t s = c10::hip::getCurrentHIPStream().stream();
  std::vector<Tensor> keep;
  Batch<1> batch[3];
  int blocks = 0;
  for (int k = 0; k < 3; ++k) {
    for (const Tensor& t : tensors) {
      if (t.scalar_type() != TYPES[k] || t.numel() == 0) continue;
      Item<1> e{};
      if (!as_rows<1>({&t}, &e)) {
        keep.push_back(t.contiguous());
        e = must<1>({&keep.back()});
      }
      batch[k].add(e, {(long)t.element_size()});
    }
    batch[k].group(16 / (TYPES[k] == at::kFloat ? 4 : 2));
    blocks += batch[k].blocks();
  }
  const auto f32 = tensors[0].options().dtype(at::kFloat);
  Tensor result = at::empty({2}, f32);
  Tensor sums = at::empty({std::max(blocks, 1)}, f32.dtype(at::kDouble));
  double* at_sums = sums.data_ptr<double>();
  auto kinds = [&](auto f) {
    if (kind == SQUARES) {
      f(std::integral_constant<int, SQUARES>());
    } else if (kind == ABSOLUTES) {
      f(std::integral_constant<int, ABSOLUTES>());
    } else {
      f(std::integral_constant<int, LARGEST>());
    }
  };
  kinds([&](auto c) {
    constexpr int K = decltype(c)::value;
    for (int k = 0; k < 3; ++k) {
      by_type(TYPES[k], [&](auto* p) {
        using T = std::remove_pointer_t<decltype(p)>;
        batch[k].launch([&](const List<1>& list, int b) {
          norm_kernel<T, K><<<b, THREADS, 0, s>>>(list, at_sums);
          check_hip(hipGetLastError());
          at_sums += b;
        });
      });
    }
    norm_end_kernel<K><<<1, 1024, 0, s>>>(
        sums.data_ptr<double>(), blocks, max_norm, result.data_ptr<float>());
    check_hip(hipGetLastError());
  });
  if (out) scale_pass(tensors, *out, result.data_ptr<float>(), s);
  return result;
}

// -> nu; writes out
Tensor trust_region(std::vector<Tensor> updates, std::vector<Tensor> grads,
                    std::vector<Tensor> out, double lr, double kl) {
  TORCH_CHECK_VALUE(!updates.empty(), "kl_clip: no tensors");
  check_lists("kl_clip", {&updates, &grads, &out});
  check_outputs("kl_clip", updates, out);
  const c10::OptionalDeviceGuard guard(updates[0].device());
  const hipStream_t s = c10::hip::getCurrentHIPStream().stream();
  std::vector<Tensor> keep;
  Batch<2> batch[9];
  int blocks = 0;
  for (int k = 0; k < 9; ++k) {
    const at::ScalarType tu = TYPES[k / 3], tg = TYPES[k % 3];
    for (size_t i = 0; i < updates.size(); ++i) {
      if (updates[i].scalar_type() != tu || grads[i].scalar_type() != tg ||
          updates[i].numel() == 0) {
        continue;
      }
      Item<2> e{};
      if (other_sign(updates[i], grads[i]) ||
          !as_rows<2>({&updates[i], &grads[i]}, &e)) {
        keep.push_back(updates[i].resolve_neg().contiguous());
        keep.push_back(grads[i].resolve_neg().contiguous());
        e = must<2>({&keep[keep.size() - 2], &keep.back()});
      }
      batch[k].add(e, {(long)updates[i].element_size(),
                       (long)grads[i].element_size()});
    }
    batch[k].group(16 / (tu == at::kFloat ? 4 : 2));
    blocks += batch[k].blocks();
  }
  const auto f32 = updates[0].options().dtype(at::kFloat);
  Tensor result = at::empty({2}, f32);
  Tensor sums = at::empty({std::max(blocks, 1)}, f32.dtype(at::kDouble));
  double* at_sums = sums.data_ptr<double>();
  for (int k = 0; k < 9; ++k) {
    if (batch[k].items.empty()) continue;
    by_type(TYPES[k / 3], [&](auto* pu) {
      using U = std::remove_pointer_t<decltype(pu)>;
      by_type(TYPES[k % 3], [&](auto* pg) {
        using G = std::remove_pointer_t<decltype(pg)>;
        batch[k].launch([&](const List<2>& list, int b) {
          dot_kernel<U, G><<<b, THREADS, 0, s>>>(list, at_sums);
          check_hip(hipGetLastError());
          at_sums += b;
        });
      });
    });
  }
  trust_end_kernel<<<1, 1024, 0, s>>>(sums.data_ptr<double>(), blocks, lr, kl,
                                      result.data_ptr<float>());
  check_hip(hipGetLastError());
  scale_pass(updates, out, result.data_ptr<float>(), s);
  return result.select(0, 0);
}
