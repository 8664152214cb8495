// Cross entropy of a vocabulary projection, and its gradients, without the
// logits in memory.
//
//   z[n, v]  = sum_d x[n, d] w[v, d] + b[v]
//   lse[n]   = log sum_v exp z[n, v]
//   loss[n]  = lse[n] - (1 - eps) z[n, t_n] - eps / V sum_v z[n, v]
//   g[n, v]  = c_n (exp(z[n, v] - lse[n]) - (1 - eps) [v = t_n] - eps / V)
//   dx = g w,   dw = g^T x,   db = sum_n g,    c_n = d(total) / d(loss[n])
//
// Forward: a workgroup makes one tile of z in registers and leaves, for each
// of its rows n, the tile's maximum, the sum of exp(z - maximum) and (with
// smoothed labels) the sum of z; a wave per row joins the tiles.  Backward:
// piece by piece of the vocabulary, z is made once more, turned into g in
// registers and written in the inputs' type, then multiplied with w and x.
//
// Rows that the loss leaves out (ignore_index) are dropped before the first
// product: x is packed to the kept rows, so padding costs nothing and what it
// holds (infinities, NaN) reaches no sum.
#include "tile_mfma.h"
#include "vocab_loss.h"

#include <algorithm>
#include <cmath>

namespace vocab_loss {
namespace {

using tile::f32x4;
using tile::Shape;

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float LN2 = 0.69314718055994530942f;

// ------------------------------------------------------------ small helpers
template <class T>
__device__ __forceinline__ float to_float(T v) {
  return (float)v;
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) v += __shfl_xor(v, s);
  return v;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) v = fmaxf(v, __shfl_xor(v, s));
  return v;
}

// a maximum to subtract: -inf (nothing seen, or all of it -inf) gives 0, so
// that exp(-inf - 0) is 0 and a NaN still shows in the sum
__device__ __forceinline__ float safe(float m) {
  return m == -INFINITY ? 0.f : m;
}

// ------------------------------------------------------- kept rows, one block
// pos[n]: the row's place among the kept ones, or -1; idx, tgt: the kept rows'
// numbers and targets, BAD for a target outside [0, vocab).
constexpr int SCAN = 1024;

template <class I>
__global__ __launch_bounds__(SCAN) void scan_kernel(
    const I* __restrict__ target, long rows, long ignore, long vocab,
    int* __restrict__ pos, int* __restrict__ idx, int* __restrict__ tgt,
    int* __restrict__ count) {
  __shared__ int sums[SCAN / 64];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  int done = 0;
  for (long base = 0; base < rows; base += SCAN) {
    const long n = base + t;
    const long v = n < rows ? (long)target[n] : ignore;
    const bool keep = n < rows && v != ignore;
    const unsigned long long mask = __ballot(keep);
    if (lane == 0) sums[wave] = __popcll(mask);
    __syncthreads();
    int before = done, all = 0;
#pragma unroll
    for (int w = 0; w < SCAN / 64; ++w) {
      const int s = sums[w];
      before += w < wave ? s : 0;
      all += s;
    }
    const int at = before + __popcll(mask & ((1ull << lane) - 1));
    if (n < rows) pos[n] = keep ? at : -1;
    if (keep) {
      idx[at] = (int)n;
      tgt[at] = (v >= 0 && v < vocab) ? (int)v : BAD;
    }
    done += all;
    __syncthreads();
  }
  if (t == 0) *count = done;
}

// ------------------------------------------------------------------ packing
// out[i, :] = in[idx ? idx[i] : i, :], zeros from `cols` to `ldo`
template <class T>
__global__ void pack_kernel(const T* __restrict__ in, long ld, long step,
                            long rows, int cols, const int* __restrict__ idx,
                            const int* __restrict__ count,
                            T* __restrict__ out, int ldo, int wide) {
  const long have = count ? *count : rows;
  constexpr int E = 16 / sizeof(T);
  using V = __attribute__((ext_vector_type(4))) int;
  const int chunks = ldo / E;
  const long total = have * chunks;
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += (long)gridDim.x * blockDim.x) {
    const long r = i / chunks;
    const int c = (int)(i - r * chunks) * E;
    const long from = idx ? idx[r] : r;
    const T* p = in + from * ld;
    V v;
    if (wide) {
      v = *reinterpret_cast<const V*>(p + c);
    } else {
      T e[E];
#pragma unroll
      for (int j = 0; j < E; ++j) {
        e[j] = c + j < cols ? p[(long)(c + j) * step] : (T)0.f;
      }
      __builtin_memcpy(&v, e, 16);
    }
    *reinterpret_cast<V*>(out + r * ldo + c) = v;
  }
}

// -------------------------------------------------------------- logits tiles
// Rows of the tile are vocabulary entries, columns are tokens: a lane then
// holds 4 neighbouring entries of one token, which it can write at once, and
// a token's sums stay within a column.
template <class T, class S>
__global__ __launch_bounds__(S::THREADS) void stats_kernel(
    const T* __restrict__ w, long ldw, const T* __restrict__ x, long ldx,
    const T* __restrict__ bias, int vocab, int dim, const int* count, int mt,
    int nt, const int* __restrict__ tgt, int smooth,
    float* __restrict__ pmax, float* __restrict__ psum,
    float* __restrict__ pz, float* __restrict__ ztgt) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  int tm, tn;
  tile::pick(blockIdx.x, mt, nt, &tm, &tn);
  const int rows = *count;
  const int m0 = tm * S::BM, n0 = tn * S::BN;
  if (n0 >= rows) return;
  f32x4 acc[S::MI][S::NI] = {};
  tile::product<T, false, false, S>(w, ldw, m0, vocab, x, ldx, n0, rows, 0,
                                    dim, dim, smem, acc);

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int i = lane & 15, g = lane >> 4;
  const int wrow = (wave / S::WN) * (S::MI * 16);
  const int wcol = (wave % S::WN) * (S::NI * 16);
  float mx[S::NI], sm[S::NI], zs[S::NI];
  int t[S::NI];
#pragma unroll
  for (int ni = 0; ni < S::NI; ++ni) {
    const int n = n0 + wcol + ni * 16 + i;
    t[ni] = n < rows ? tgt[n] : BAD;
    mx[ni] = -INFINITY;
    sm[ni] = 0.f;
    zs[ni] = 0.f;
  }
#pragma unroll
  for (int mi = 0; mi < S::MI; ++mi) {
    const int v = m0 + wrow + mi * 16 + g * 4;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const bool in = v + r < vocab;
      const float b = bias && in ? to_float(bias[v + r]) : 0.f;
#pragma unroll
      for (int ni = 0; ni < S::NI; ++ni) {
        const float z = acc[mi][ni][r] + b;
        if (v + r == t[ni] && in) ztgt[n0 + wcol + ni * 16 + i] = z;
        zs[ni] += in ? z : 0.f;
        acc[mi][ni][r] = in ? z : -INFINITY;
        mx[ni] = fmaxf(mx[ni], acc[mi][ni][r]);
      }
    }
  }
  float* red = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int ni = 0; ni < S::NI; ++ni) {
    mx[ni] = fmaxf(mx[ni], __shfl_xor(mx[ni], 16));
    mx[ni] = fmaxf(mx[ni], __shfl_xor(mx[ni], 32));
    const float m = safe(mx[ni]);
#pragma unroll
    for (int mi = 0; mi < S::MI; ++mi) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        sm[ni] += __builtin_amdgcn_exp2f((acc[mi][ni][r] - m) * LOG2E);
      }
    }
    sm[ni] += __shfl_xor(sm[ni], 16);
    sm[ni] += __shfl_xor(sm[ni], 32);
    zs[ni] += __shfl_xor(zs[ni], 16);
    zs[ni] += __shfl_xor(zs[ni], 32);
    if (g == 0) {
      float* p = red + ((wave / S::WN) * S::BN + wcol + ni * 16 + i) * 3;
      p[0] = mx[ni];
      p[1] = sm[ni];
      p[2] = zs[ni];
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < S::BN; c += S::THREADS) {
    if (n0 + c >= rows) continue;
    float m = -INFINITY, s = 0.f, z = 0.f;
#pragma unroll
    for (int k = 0; k < S::WM; ++k) m = fmaxf(m, red[(k * S::BN + c) * 3]);
#pragma unroll
    for (int k = 0; k < S::WM; ++k) {
      const float* p = red + (k * S::BN + c) * 3;
      s += p[1] * __builtin_amdgcn_exp2f((safe(p[0]) - safe(m)) * LOG2E);
      z += p[2];
    }
    const long at = (long)(n0 + c) * mt + tm;
    pmax[at] = m;
    psum[at] = s;
    if (smooth) pz[at] = z;
  }
}

// one wave per row of the call: joins the tiles' sums
__global__ __launch_bounds__(256) void join_kernel(
    const float* __restrict__ pmax, const float* __restrict__ psum,
    const float* __restrict__ pz, const float* __restrict__ ztgt,
    const int* __restrict__ pos, const int* __restrict__ tgt, long rows,
    int mt, float eps, float share, float* __restrict__ lse,
    float* __restrict__ loss) {
  const int lane = threadIdx.x & 63;
  const long n = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (n >= rows) return;
  const int p = pos[n];
  if (p < 0) {
    if (lane == 0) loss[n] = 0.f;
    return;
  }
  const long at = (long)p * mt;
  float m = -INFINITY;
  for (int k = lane; k < mt; k += 64) m = fmaxf(m, pmax[at + k]);
  m = wave_max(m);
  const float base = safe(m);
  float s = 0.f, z = 0.f;
  for (int k = lane; k < mt; k += 64) {
    s += psum[at + k] *
         __builtin_amdgcn_exp2f((safe(pmax[at + k]) - base) * LOG2E);
    if (eps != 0.f) z += pz[at + k];
  }
  s = wave_sum(s);
  z = wave_sum(z);
  if (lane == 0) {
    const float l = base + __builtin_amdgcn_logf(s) * LN2;
    lse[p] = l;
    float v = l - (1.f - eps) * ztgt[p];
    if (eps != 0.f) v -= share * z;
    loss[n] = tgt[p] == BAD ? NAN : v;
  }
}

// one block, in a fixed order: total = sum of loss (/ count for the mean)
__global__ __launch_bounds__(1024) void total_kernel(
    const float* __restrict__ loss, long rows, const int* __restrict__ count,
    int mean, float* __restrict__ total) {
  __shared__ double part[16];
  double s = 0.0;
  for (long n = threadIdx.x; n < rows; n += 1024) s += (double)loss[n];
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) s += __shfl_xor(s, k);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int k = 0; k < 16; ++k) t += part[k];
    *total = (float)(mean ? t / (double)*count : t);
  }
}

// ---------------------------------------------------------- row coefficients
// coef[i] = d(total)/d(loss of kept row i) times a power of two, scale[0];
// scale[1] is its inverse.  fp16 holds g to 6e-8 only, and c_n = 1/rows times
// a small probability is soon below that: there the largest |c_n| is brought
// to [2^14, 2^15) (|g| <= |c_n|, and the type ends at 65504) and the products
// are scaled back in fp32.
__global__ __launch_bounds__(1024) void coef_kernel(
    const float* __restrict__ up, int each, int mean,
    const int* __restrict__ idx, const int* __restrict__ tgt,
    const int* __restrict__ count, int lift, float* __restrict__ coef,
    float* __restrict__ scale) {
  __shared__ float part[16];
  __shared__ float shared_scale;
  const int rows = *count;
  const float one = each ? 1.f : (mean ? *up / (float)rows : *up);
  float top = 0.f;
  if (lift) {
    if (each) {
      for (int i = threadIdx.x; i < rows; i += 1024) {
        const float a = fabsf(up[idx[i]]);
        if (a < INFINITY) top = fmaxf(top, a);
      }
    } else {
      top = fabsf(one) < INFINITY ? fabsf(one) : 0.f;
    }
    top = wave_max(top);
  }
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    float m = 0.f;
    for (int k = 0; k < 16; ++k) m = fmaxf(m, part[k]);
    int e = 0;
    if (m > 0.f) {
      e = 14 - (int)floorf(__builtin_amdgcn_logf(m));
      e = e > 100 ? 100 : (e < -100 ? -100 : e);
    }
    shared_scale = ldexpf(1.f, e);
    scale[0] = shared_scale;
    scale[1] = ldexpf(1.f, -e);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows; i += 1024) {
    const float c = (each ? up[idx[i]] : one) * shared_scale;
    coef[i] = tgt[i] == BAD ? NAN : c;
  }
}

// ------------------------------------------------------------ gradient tiles
// g[n, v - v0] for a piece [v0, v0 + piece) of the vocabulary; entries from
// the piece's end to ldg are zeros.  The bias gradient's part of a tile is
// summed before the rounding.
template <class T, class S>
__global__ __launch_bounds__(S::THREADS) void grad_kernel(
    const T* __restrict__ w, long ldw, const T* __restrict__ x, long ldx,
    const T* __restrict__ bias, int v0, int piece, int dim, const int* count,
    int mt, int nt, const int* __restrict__ tgt,
    const float* __restrict__ lse, const float* __restrict__ coef, float eps,
    float share, T* __restrict__ grad, long ldg, float* __restrict__ pbias,
    long vocab) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  int tm, tn;
  tile::pick(blockIdx.x, mt, nt, &tm, &tn);
  const int rows = *count;
  const int m0 = tm * S::BM, n0 = tn * S::BN;
  if (n0 >= rows) return;
  f32x4 acc[S::MI][S::NI] = {};
  tile::product<T, false, false, S>(w + (long)v0 * ldw, ldw, m0, piece, x,
                                    ldx, n0, rows, 0, dim, dim, smem, acc);

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int i = lane & 15, g = lane >> 4;
  const int wrow = (wave / S::WN) * (S::MI * 16);
  const int wcol = (wave % S::WN) * (S::NI * 16);
  float l[S::NI], c[S::NI];
  int t[S::NI];
#pragma unroll
  for (int ni = 0; ni < S::NI; ++ni) {
    const int n = n0 + wcol + ni * 16 + i;
    const bool in = n < rows;
    l[ni] = in ? lse[n] : 0.f;
    c[ni] = in ? coef[n] : 0.f;
    t[ni] = in ? tgt[n] - v0 : BAD;
  }
  float* red = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int mi = 0; mi < S::MI; ++mi) {
    const int vl = wrow + mi * 16 + g * 4;  // within the tile
    const int v = m0 + vl;                  // within the piece
    float b[4], sb[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      b[r] = bias && v + r < piece ? to_float(bias[v0 + v + r]) : 0.f;
    }
#pragma unroll
    for (int ni = 0; ni < S::NI; ++ni) {
      const int n = n0 + wcol + ni * 16 + i;
      T out[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float p =
            __builtin_amdgcn_exp2f((acc[mi][ni][r] + b[r] - l[ni]) * LOG2E);
        float d = p - share;
        if (v + r == t[ni]) d -= 1.f - eps;
        d *= c[ni];
        d = v + r < piece ? d : 0.f;
        sb[r] += n < rows ? d : 0.f;
        out[r] = (T)d;
      }
      if (n < rows && v < ldg) {
        __builtin_memcpy(grad + (long)n * ldg + v, out, 4 * sizeof(T));
      }
    }
    if (pbias) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float s = sb[r];
        s += __shfl_xor(s, 1);
        s += __shfl_xor(s, 2);
        s += __shfl_xor(s, 4);
        s += __shfl_xor(s, 8);
        if (i == 0) red[(wave % S::WN) * S::BM + vl + r] = s;
      }
    }
  }
  if (pbias) {
    __syncthreads();
    for (int k = threadIdx.x; k < S::BM; k += S::THREADS) {
      if (m0 + k >= piece) continue;
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < S::WN; ++j) s += red[j * S::BM + k];
      pbias[(long)tn * vocab + v0 + m0 + k] = s;
    }
  }
}

template <class T>
__global__ void bias_kernel(const float* __restrict__ pbias, long vocab,
                            int bn, const int* __restrict__ count,
                            const float* __restrict__ scale,
                            T* __restrict__ out) {
  const long v = (long)blockIdx.x * blockDim.x + threadIdx.x;
  if (v >= vocab) return;
  const int parts = (*count + bn - 1) / bn;
  float s = 0.f;
  for (int k = 0; k < parts; ++k) s += pbias[(long)k * vocab + v];
  out[v] = (T)(s * scale[1]);
}

// ------------------------------------------------------------- dx += g w
// Rows of the tile are hidden units, columns tokens, k the piece's entries,
// cut into `splits` runs of `run` values that add to slabs of their own.
template <class T, class S>
__global__ __launch_bounds__(S::THREADS) void dx_kernel(
    const T* __restrict__ w, long ldw, const T* __restrict__ grad, long ldg,
    int piece, int dim, const int* count, int mt, int nt, int run, int first,
    float* __restrict__ slabs, long slab) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int split = blockIdx.x / (mt * nt);
  int tm, tn;
  tile::pick(blockIdx.x - split * mt * nt, mt, nt, &tm, &tn);
  const int rows = *count;
  const int m0 = tm * S::BM, n0 = tn * S::BN;
  if (n0 >= rows) return;
  const int kbeg = split * run;
  const int kend = (int)ldg - kbeg < run ? (int)ldg : kbeg + run;
  f32x4 acc[S::MI][S::NI] = {};
  tile::product<T, true, false, S>(w, ldw, m0, dim, grad, ldg, n0, rows, kbeg,
                                   kend, piece, smem, acc);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int i = lane & 15, g = lane >> 4;
  float* out = slabs + split * slab;
#pragma unroll
  for (int mi = 0; mi < S::MI; ++mi) {
    const int d = m0 + (wave / S::WN) * (S::MI * 16) + mi * 16 + g * 4;
    if (d >= dim) continue;  // dim is a multiple of 4
#pragma unroll
    for (int ni = 0; ni < S::NI; ++ni) {
      const int n = n0 + (wave % S::WN) * (S::NI * 16) + ni * 16 + i;
      if (n >= rows) continue;
      f32x4* p = reinterpret_cast<f32x4*>(out + (long)n * dim + d);
      *p = first ? acc[mi][ni] : *p + acc[mi][ni];
    }
  }
}

// dx of every row of the call: the slabs' sum, or zeros for a row left out
template <class T>
__global__ void dx_out_kernel(const float* __restrict__ slabs, long slab,
                              int splits, int ldim, int dim, long rows,
                              const int* __restrict__ pos,
                              const float* __restrict__ scale,
                              T* __restrict__ out) {
  const float inv = scale[1];
  const long total = rows * dim;
  for (long k = (long)blockIdx.x * blockDim.x + threadIdx.x; k < total;
       k += (long)gridDim.x * blockDim.x) {
    const long n = k / dim;
    const int d = (int)(k - n * dim);
    const int p = pos[n];
    float s = 0.f;
    if (p >= 0) {
      for (int j = 0; j < splits; ++j) s += slabs[j * slab + (long)p * ldim + d];
    }
    out[k] = (T)(s * inv);
  }
}

// ------------------------------------------------------------- dw = g^T x
// Rows of the tile are hidden units, columns vocabulary entries, k tokens.
template <class T, class S>
__global__ __launch_bounds__(S::THREADS) void dw_kernel(
    const T* __restrict__ x, long ldx, const T* __restrict__ grad, long ldg,
    int piece, int dim, int ldim, const int* count, int mt, int nt, int run,
    const float* __restrict__ scale, T* __restrict__ out,
    float* __restrict__ slabs, long slab) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int split = blockIdx.x / (mt * nt);
  int tm, tn;
  tile::pick(blockIdx.x - split * mt * nt, mt, nt, &tm, &tn);
  const int rows = *count;
  const int m0 = tm * S::BM, n0 = tn * S::BN;
  const int kbeg = split * run;
  const int kend = rows - kbeg < run ? rows : kbeg + run;
  f32x4 acc[S::MI][S::NI] = {};
  tile::product<T, true, true, S>(x, ldx, m0, ldim, grad, ldg, n0,
                                  (int)ldg, kbeg, kend, kend, smem, acc);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int i = lane & 15, g = lane >> 4;
  const float inv = scale[1];
#pragma unroll
  for (int mi = 0; mi < S::MI; ++mi) {
    const int d = m0 + (wave / S::WN) * (S::MI * 16) + mi * 16 + g * 4;
#pragma unroll
    for (int ni = 0; ni < S::NI; ++ni) {
      const int v = n0 + (wave % S::WN) * (S::NI * 16) + ni * 16 + i;
      if (v >= piece || d >= dim) continue;
      if (slabs) {
        float* p = slabs + split * slab + (long)v * ldim + d;
        *reinterpret_cast<f32x4*>(p) = acc[mi][ni];
      } else if (dim % 4 == 0) {
        T o[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = (T)(acc[mi][ni][r] * inv);
        __builtin_memcpy(out + (long)v * dim + d, o, 4 * sizeof(T));
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (d + r < dim) out[(long)v * dim + d + r] = (T)(acc[mi][ni][r] * inv);
        }
      }
    }
  }
}

template <class T>
__global__ void dw_out_kernel(const float* __restrict__ slabs, long slab,
                              int splits, int ldim, int dim, long entries,
                              const float* __restrict__ scale,
                              T* __restrict__ out) {
  const float inv = scale[1];
  const long total = entries * dim;
  for (long k = (long)blockIdx.x * blockDim.x + threadIdx.x; k < total;
       k += (long)gridDim.x * blockDim.x) {
    const long v = k / dim;
    const int d = (int)(k - v * dim);
    float s = 0.f;
    for (int j = 0; j < splits; ++j) s += slabs[j * slab + v * ldim + d];
    out[k] = (T)(s * inv);
  }
}

int blocks_for(long work) {
  return (int)std::min<long>(std::max<long>((work + 255) / 256, 1), 8192);
}

int ceil_div(long a, long b) { return (int)((a + b - 1) / b); }

using Wide = Shape<256, 256, 2, 4>;
using Mid = Shape<128, 128, 2, 2>;

template <class F>
void with_lds(F* kernel, int bytes) {
  check(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                            hipFuncAttributeMaxDynamicSharedMemorySize,
                            bytes));
}

template <class T>
struct Run {
  template <class S>
  static void stats(const Forward& f, hipStream_t s) {
    const int mt = ceil_div(f.vocab, S::BM), nt = ceil_div(f.rows, S::BN);
    with_lds(stats_kernel<T, S>, S::LDS);
    stats_kernel<T, S><<<mt * nt, S::THREADS, S::LDS, s>>>(
        (const T*)f.w, f.ldw, (const T*)f.x, f.ldx, (const T*)f.bias,
        (int)f.vocab, f.ldx, f.count, mt, nt, f.tgt, f.eps != 0.f, f.pmax,
        f.psum, f.pz, f.ztgt);
    check(hipGetLastError());
    join_kernel<<<ceil_div(f.rows, 4), 256, 0, s>>>(
        f.pmax, f.psum, f.pz, f.ztgt, f.pos, f.tgt, f.rows, mt, f.eps,
        f.eps / (float)f.vocab, f.lse, f.loss);
    check(hipGetLastError());
  }

  template <class S>
  static void pieces(const Backward& b, hipStream_t s) {
    const int dim = b.ldx;
    const int nt = ceil_div(b.rows, S::BN), md = ceil_div(dim, S::BM);
    const long slab = b.rows * dim;
    with_lds(grad_kernel<T, S>, S::LDS);
    with_lds(dx_kernel<T, S>, S::LDS);
    with_lds(dw_kernel<T, S>, S::LDS);
    for (long v0 = 0; v0 < b.vocab; v0 += b.piece) {
      const int piece = (int)std::min(b.piece, b.vocab - v0);
      const long ldg = (piece + 7) / 8 * 8;
      const int mt = ceil_div(piece, S::BM);
      grad_kernel<T, S><<<mt * nt, S::THREADS, S::LDS, s>>>(
          (const T*)b.w, b.ldw, (const T*)b.x, b.ldx, (const T*)b.bias,
          (int)v0, piece, dim, b.count, mt, nt, b.tgt, b.lse, b.coef, b.eps,
          b.eps / (float)b.vocab, (T*)b.grad, ldg, b.pbias, b.vocab);
      check(hipGetLastError());
      if (b.dx) {
        const int run = ceil_div(ceil_div(ldg, b.dx_splits), 64) * 64;
        dx_kernel<T, S><<<md * nt * b.dx_splits, S::THREADS, S::LDS, s>>>(
            (const T*)b.w + v0 * b.ldw, b.ldw, (const T*)b.grad, ldg, piece,
            dim, b.count, md, nt, run, v0 == 0, b.dx_slabs, slab);
        check(hipGetLastError());
      }
      if (b.dw) {
        const int vt = ceil_div(piece, S::BN);
        const int run = ceil_div(ceil_div(b.rows, b.dw_splits), 64) * 64;
        T* out = (T*)b.dw + v0 * b.dim;
        const long part = (long)piece * dim;
        dw_kernel<T, S><<<md * vt * b.dw_splits, S::THREADS, S::LDS, s>>>(
            (const T*)b.x, b.ldx, (const T*)b.grad, ldg, piece, b.dim, dim,
            b.count, md, vt, run, b.scale, out,
            b.dw_splits > 1 ? b.dw_slabs : nullptr, part);
        check(hipGetLastError());
        if (b.dw_splits > 1) {
          dw_out_kernel<T><<<blocks_for((long)piece * b.dim), 256, 0, s>>>(
              b.dw_slabs, part, b.dw_splits, dim, b.dim, piece, b.scale, out);
          check(hipGetLastError());
        }
      }
    }
    if (b.dx) {
      dx_out_kernel<T><<<blocks_for(b.rows * b.dim), 256, 0, s>>>(
          b.dx_slabs, slab, b.dx_splits, dim, b.dim, b.rows, b.pos, b.scale,
          (T*)b.dx);
      check(hipGetLastError());
    }
    if (b.db) {
      bias_kernel<T><<<ceil_div(b.vocab, 256), 256, 0, s>>>(
          b.pbias, b.vocab, S::BN, b.count, b.scale, (T*)b.db);
      check(hipGetLastError());
    }
  }
};

template <class F>
void by_type(Type t, F f) {
  switch (t) {
    case Type::bf16: f((__bf16*)nullptr); break;
    case Type::fp16: f((_Float16*)nullptr); break;
    case Type::fp32: f((float*)nullptr); break;
  }
}

// Wide tiles do twice the work per byte that goes through LDS and take a CU
// each; they pay once they fill the card.
bool wide(long m, long n) {
  return (long)ceil_div(m, 256) * ceil_div(n, 256) >= 256;
}

}  // namespace

Plan plan(long rows, long vocab, int ldim, int size) {
  Plan p;
  p.wide = wide(vocab, rows);
  p.edge = p.wide ? 256 : 128;
  p.tiles = ceil_div(vocab, p.edge);
  p.row_tiles = ceil_div(rows, p.edge);
  // a piece of the vocabulary: 256 MB of g at most, which the card's last
  // cache then holds between the three products; offsets within a tile of g
  // stay below 2^31 for rows of up to a million entries
  const long most = std::min<long>(
      std::max<long>((256l << 20) / (rows * size), p.edge), 1l << 20);
  p.piece = std::min(vocab, most / p.edge * p.edge);
  const long dx_tiles = (long)ceil_div(ldim, p.edge) * p.row_tiles;
  const long dw_tiles =
      (long)ceil_div(ldim, p.edge) * ceil_div(p.piece, p.edge);
  const long want = p.wide ? 256 : 512;
  p.dx_splits = (int)std::max<long>(
      1, std::min<long>({want / dx_tiles, p.piece / 512, 64}));
  p.dw_splits = (int)std::max<long>(
      1, std::min<long>({want / dw_tiles, rows / 512, 16}));
  return p;
}

void scan(const void* target, bool wide_ints, long rows, long ignore,
          long vocab, int* pos, int* idx, int* tgt, int* count,
          hipStream_t s) {
  if (wide_ints) {
    scan_kernel<long><<<1, SCAN, 0, s>>>((const long*)target, rows, ignore,
                                         vocab, pos, idx, tgt, count);
  } else {
    scan_kernel<int><<<1, SCAN, 0, s>>>((const int*)target, rows, ignore,
                                        vocab, pos, idx, tgt, count);
  }
  check(hipGetLastError());
}

void pack(Type t, const void* in, long ld, long step, long rows, int cols,
          const int* idx, const int* count, void* out, int ldo,
          hipStream_t s) {
  by_type(t, [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    const bool wide_loads = step == 1 && ldo == cols &&
                            (uintptr_t)in % 16 == 0 &&
                            ld * sizeof(T) % 16 == 0;
    pack_kernel<T><<<blocks_for(rows * (ldo * sizeof(T) / 16)), 256, 0, s>>>(
        (const T*)in, ld, step, rows, cols, idx, count, (T*)out, ldo,
        wide_loads);
    check(hipGetLastError());
  });
}

void forward(Type t, const Forward& f, hipStream_t s) {
  by_type(t, [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    if (f.plan.wide) {
      Run<T>::template stats<Wide>(f, s);
    } else {
      Run<T>::template stats<Mid>(f, s);
    }
  });
}

void total(const float* loss, long rows, const int* count, bool mean,
           float* out, hipStream_t s) {
  total_kernel<<<1, 1024, 0, s>>>(loss, rows, count, mean, out);
  check(hipGetLastError());
}

void backward(Type t, const Backward& b, hipStream_t s) {
  coef_kernel<<<1, 1024, 0, s>>>(b.up, b.each, b.mean, b.idx, b.tgt, b.count,
                                 t == Type::fp16, b.coef, b.scale);
  check(hipGetLastError());
  by_type(t, [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    if (b.plan.wide) {
      Run<T>::template pieces<Wide>(b, s);
    } else {
      Run<T>::template pieces<Mid>(b, s);
    }
  });
}

}  // namespace vocab_loss
