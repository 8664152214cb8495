// Cross entropy of a vocabulary projection, and its gradients, without the
// logits in memory.
//
//   z[n, v]  = sum_d x[n, d] w[v, d] + b[v]
//   lse[n]   = log sum_v exp z[n, v]
//   loss[n]  = lse[n] - (1 - eps) z[n, t_n] - eps / V sum_v z[n, v]
//   g[n, v]  = c_n (exp(z[n, v] - lse[n]) - (1 - eps) [v = t_n] - eps / V)
//   dx = g w,   dw = g^T x,   db = sum_n g,    c_n = d(total) / d(loss[n])
//
// A workgroup makes one tile of z in registers.  Of each band of its rows it
// leaves, for every token n, the band's largest z, the sum of exp(z - largest)
// (the powers) and, with smoothed labels, the sum of z; a wave per row joins
// them.  The difference is taken before it is scaled for exp2: one fused
// multiply-add instead would be off by the rounding of largest * log2(e), a
// factor of 2^64 where a mask adds -1e9 to a whole band.
//
// Gradients, either of two ways:
//   kept: the forward pass writes the powers themselves, in 16 bits for 16-bit
//     inputs; once the sums are joined a pass over them makes g, and g is multiplied
//     with w and x: 3 products in all.  They exist during the call only; what
//     is kept for the backward pass are the gradients for an upstream factor
//     of 1.
//   again: the backward pass makes z once more, piece by piece of the
//     vocabulary: 4 products, and a piece's g at a time.  For losses of single
//     rows, whose factors come with the backward pass, and where the powers
//     would take too much memory.
// g is rounded to the inputs' type once before the products, as it would be by
// a layer that computes in that type; kept powers are rounded to fp16 before
// that (fp32 inputs: fp32).  The target's own entry is always made from fp32:
// there p - 1 cancels.
//
// Rows that the loss leaves out (ignore_index) are dropped before the first
// product: x is packed to the kept rows, so padding costs nothing and what it
// holds (infinities, NaN) reaches no sum.
#include "tile_mfma.h"
#include "vocab_loss.h"

#include <algorithm>
#include <atomic>
#include <cmath>

namespace vocab_loss {
namespace {

using tile::f32x4;
using tile::Shape;

constexpr float LOG2E = 1.44269504088896340736f;

// ------------------------------------------------------------ small helpers
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

// a reference to subtract: -inf (nothing seen, or all of it -inf) gives 0, so
// that exp2(-inf - 0) is 0 and a NaN still shows in the sum
__device__ __forceinline__ float safe(float m) {
  return m == -INFINITY ? 0.f : m;
}

__device__ __forceinline__ float power(float z, float m) {
  return __builtin_amdgcn_exp2f((z - m) * LOG2E);
}

// The type that powers are kept in: 16 bits are best used as fp16, also for
// bf16 (without the lift below, gradients off by 2.1e-3 of their norm instead
// of 2.6e-3).  A power is at most 1; times 2^15, those down to 2^-29 of a
// band's largest keep all 11 bits.
template <class T>
using Power = std::conditional_t<sizeof(T) == 2, _Float16, float>;
template <class T>
constexpr float LIFT = sizeof(T) == 2 ? 32768.f : 1.f;

// ------------------------------------------------------- kept rows, one block
// pos[n]: the row's place among the kept ones, or -1; idx, tgt: the kept rows'
// numbers and targets, BAD for a target outside [0, vocab).
constexpr int SCAN = 1024;   // threads
constexpr int EACH = 8;      // targets of a thread in flight

template <class I>
__global__ __launch_bounds__(SCAN) void scan_kernel(
    const I* __restrict__ target, long rows, long ignore, long vocab,
    int* __restrict__ pos, int* __restrict__ idx, int* __restrict__ tgt,
    int* __restrict__ count) {
  constexpr int WAVES = SCAN / 64, PARTS = WAVES * EACH;  // 128 counts
  __shared__ int sums[PARTS];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  int done = 0;
  for (long base = 0; base < rows; base += SCAN * EACH) {
    long v[EACH];
    unsigned long long mask[EACH];
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      const long n = base + k * SCAN + t;
      v[k] = n < rows ? (long)target[n] : ignore;
    }
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      mask[k] = __ballot(v[k] != ignore);
      if (lane == 0) sums[k * WAVES + wave] = __popcll(mask[k]);
    }
    __syncthreads();
    // every wave scans the counts: exclusive sums of pairs of them
    const int a = sums[2 * lane], b = sums[2 * lane + 1];
    int s = a + b;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(s, d);
      s += lane >= d ? o : 0;
    }
    const int all = __shfl(s, 63);
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      const int part = k * WAVES + wave;
      const int end = __shfl(s, part >> 1), first = __shfl(a, part >> 1),
                second = __shfl(b, part >> 1);
      const int before =
          done + end - second - (part & 1 ? 0 : first);
      const long n = base + k * SCAN + t;
      const bool keep = v[k] != ignore;
      const int at = before + __popcll(mask[k] & ((1ull << lane) - 1));
      if (n < rows) pos[n] = keep ? at : -1;
      if (keep) {
        idx[at] = (int)n;
        tgt[at] = (v[k] >= 0 && v[k] < vocab) ? (int)v[k] : BAD;
      }
    }
    done += all;
    __syncthreads();
  }
  if (t == 0) *count = done;
}

// ------------------------------------------------------------------ packing
// How a row's values can be loaded: one by one; two 16-bit ones at a time, where
// rows begin at multiples of 4 bytes; or 16 bytes of whole and aligned rows.
enum Loads { SINGLE, PAIRS, WIDE };

// values c .. c + E of a row, zeros from `cols` on
template <class T>
__device__ __forceinline__ void copy_chunk(const T* in, long step, int c,
                                           int cols, int loads, T* out) {
  constexpr int E = 16 / sizeof(T);
  using V = __attribute__((ext_vector_type(4))) int;
  V v;
  if (loads == WIDE) {
    v = *reinterpret_cast<const V*>(in + c);
  } else if (sizeof(T) == 2 && loads == PAIRS) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = c + 2 * j;
      int pair = 0;
      if (k + 2 <= cols) {
        pair = *reinterpret_cast<const int*>(in + k);
      } else if (k < cols) {
        pair = *reinterpret_cast<const unsigned short*>(in + k);
      }
      v[j] = pair;
    }
  } else {
    T e[E];
#pragma unroll
    for (int j = 0; j < E; ++j) {
      e[j] = c + j < cols ? in[(long)(c + j) * step] : (T)0.f;
    }
    __builtin_memcpy(&v, e, 16);
  }
  *reinterpret_cast<V*>(out + c) = v;
}

// out[i, :] = in[idx ? idx[i] : i, :], zeros from `cols` to `ldo`; 2^lanes
// lanes to a row.  Bound by memory.
template <class T>
__global__ __launch_bounds__(256) void pack_kernel(
    const T* __restrict__ in, long ld, long step, long rows, int cols,
    const int* __restrict__ idx, const int* __restrict__ count,
    T* __restrict__ out, int ldo, int loads, int lanes) {
  const long have = count ? *count : rows;
  constexpr int E = 16 / sizeof(T);
  const int chunks = ldo / E, each = 1 << lanes;
  const long id = (long)blockIdx.x * 256 + threadIdx.x;
  const long all = (long)gridDim.x * 256 >> lanes;
  for (long r = id >> lanes; r < have; r += all) {
    const T* from = in + (idx ? idx[r] : r) * ld;
    for (int c = (int)id & (each - 1); c < chunks; c += each) {
      copy_chunk(from, step, c * E, cols, loads, out + r * ldo);
    }
  }
}

// Both of the above in one launch: a workgroup counts the kept rows before its
// own `prep` rows anew, numbers these and packs them.  The counting reads
// rows^2 / prep / 2 targets in all, nothing for some thousand rows (8192 rows
// of 768 in fp16: 9 us against 6 + 8 and a launch), too much for very many.
constexpr int PREP = 16;
constexpr long PREP_MOST = 16384;

template <class T, class I>
__global__ __launch_bounds__(256) void prepare_kernel(
    const I* __restrict__ target, long rows, long ignore, long vocab,
    int* __restrict__ pos, int* __restrict__ idx, int* __restrict__ tgt,
    int* __restrict__ count, const T* __restrict__ in, long ld, long step,
    int cols, T* __restrict__ out, int ldo, int loads, int prep) {
  __shared__ int part[4], from[PREP], kept;
  const int t = threadIdx.x, lane = t & 63;
  const int first = blockIdx.x * prep;
  int n = 0;
#pragma unroll 8
  for (int k = t; k < first; k += 256) n += (long)target[k] != ignore;
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) n += __shfl_xor(n, d);
  if (lane == 0) part[t >> 6] = n;
  __syncthreads();
  const int before = part[0] + part[1] + part[2] + part[3];
  if (t < 64) {
    const int r = first + t;
    const long v = t < prep && r < rows ? (long)target[r] : ignore;
    const bool keep = v != ignore;
    const unsigned long long mask = __ballot(keep);
    const int mine = __popcll(mask & ((1ull << lane) - 1));
    if (t < prep && r < rows) pos[r] = keep ? before + mine : -1;
    if (keep) {
      idx[before + mine] = r;
      tgt[before + mine] = v >= 0 && v < vocab ? (int)v : BAD;
      from[mine] = r;
    }
    if (t == 0) {
      kept = __popcll(mask);
      if (first + prep >= rows) *count = before + __popcll(mask);
    }
  }
  __syncthreads();
  constexpr int E = 16 / sizeof(T);
  const int chunks = ldo / E;
  for (int k = t; k < kept * chunks; k += 256) {
    const int r = k / chunks, c = (k - r * chunks) * E;
    copy_chunk(in + from[r] * ld, step, c, cols, loads,
               out + (long)(before + r) * ldo);
  }
}

// -------------------------------------------------------------- logits tiles
// Rows of the tile are vocabulary entries, columns are tokens: a lane then
// holds 4 neighbouring entries of one token, which it can write at once, and
// a token's sums stay within a column.  A wave's rows are one band.
// Long k: bound by the matrix cores (8192 x 30522 x 768 in fp16: 415 us at best,
// 925 TFLOP/s, 470 on the median; the library's product alone 433).  Short k: a
// tile of 256 x 256 takes 8 us besides its slices of 1.1 us, half of them the
// 65536 exponentials (8192 x 32768 x 64: one slice, 74 us for 8 rounds; with the
// powers stored 87).
struct Logits {
  long ldw;
  int ldx, v0, vocab;  // the piece [v0, v0 + vocab) of the entries
  int mt;
  const int *count, *tgt;
  // sums, KEEP
  float *pmax, *psum, *pz, *ztgt;  // [row][band]; pz null without smoothing
  int bands;
  // g, KEEP
  long ldg;
  // g
  const float *rowm, *rowi, *coef;
  float eps, share;
  float* pbias;        // [tile of tokens][entry of all]
  long all;
};

enum Mode { SUMS, KEEP, AGAIN };

template <class T, class S, int MODE>
__global__ __launch_bounds__(S::THREADS) void logits_kernel(
    const T* __restrict__ w, const T* __restrict__ x,
    const T* __restrict__ bias, T* __restrict__ grad, const Logits p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int rows = *p.count;
  int tm, tn;
  if (!tile::pick(blockIdx.x, p.mt, (rows + S::BN - 1) / S::BN, &tm, &tn)) {
    return;
  }
  const int m0 = tm * S::BM, n0 = tn * S::BN;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = lane & 15, g = lane >> 4;
  const int wrow = (wave / S::WN) * (S::MI * 16);
  const int wcol = (wave % S::WN) * (S::NI * 16);
  const int vbase = m0 + wrow + g * 4;  // + 16 mi + r
  const int nbase = n0 + wcol + i;      // + 16 ni

  int t[S::NI];
#pragma unroll
  for (int ni = 0; ni < S::NI; ++ni) {
    const int n = nbase + ni * 16;
    t[ni] = p.tgt[n < rows ? n : 0];
  }
  f32x4 acc[S::MI][S::NI];
  const auto begin = [&] {
#pragma unroll
    for (int mi = 0; mi < S::MI; ++mi) {
      f32x4 b = {};
      if (bias) {
        const int v = vbase + mi * 16;
        T t[4] = {};
        if (v + 4 <= p.vocab) {
          __builtin_memcpy(t, bias + p.v0 + v, sizeof(t));
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (v + r < p.vocab) t[r] = bias[p.v0 + v + r];
          }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) b[r] = (float)t[r];
      }
#pragma unroll
      for (int ni = 0; ni < S::NI; ++ni) acc[mi][ni] = b;
    }
  };
  tile::product<T, false, false, S>(w + (long)p.v0 * p.ldw, p.ldw, m0,
                                    p.vocab, x, p.ldx, n0, rows, 0, p.ldx,
                                    p.ldx, smem, acc, begin);

  // where a token's target is among this lane's entries: 16 mi + r, or none
#pragma unroll
  for (int ni = 0; ni < S::NI; ++ni) {
    t[ni] = nbase + ni * 16 < rows ? t[ni] - p.v0 - vbase : -1;
    if ((unsigned)t[ni] >= (unsigned)(S::MI * 16) || (t[ni] & 15) > 3 ||
        vbase + t[ni] >= p.vocab) {
      t[ni] = -1;
    }
  }
  const bool whole = m0 + S::BM <= p.vocab;
  char* stage = smem + wave * (2 * S::MI * 256 * sizeof(T));
  static_assert(S::NW * 2 * S::MI * 256 * sizeof(T) <= S::LDS, "LDS");

  if constexpr (MODE != AGAIN) {
    float zs[S::NI];
#pragma unroll
    for (int ni = 0; ni < S::NI; ++ni) {
      zs[ni] = 0.f;
      if (t[ni] >= 0) {  // selects: a branch for each entry costs 4 us of 46
        float z = 0.f;
#pragma unroll
        for (int k = 0; k < S::MI * 4; ++k) {
          z = t[ni] == (k >> 2) * 16 + (k & 3) ? acc[k >> 2][ni][k & 3] : z;
        }
        p.ztgt[nbase + ni * 16] = z;
      }
    }
    if (p.pz) {
#pragma unroll
      for (int mi = 0; mi < S::MI; ++mi) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool in = whole || vbase + mi * 16 + r < p.vocab;
#pragma unroll
          for (int ni = 0; ni < S::NI; ++ni) {
            zs[ni] += in ? acc[mi][ni][r] : 0.f;
          }
        }
      }
    }
    if (!whole) {
#pragma unroll
      for (int mi = 0; mi < S::MI; ++mi) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (vbase + mi * 16 + r >= p.vocab) {
#pragma unroll
            for (int ni = 0; ni < S::NI; ++ni) acc[mi][ni][r] = -INFINITY;
          }
        }
      }
    }
#pragma unroll
    for (int ni = 0; ni < S::NI; ++ni) {
      float m = -INFINITY;
#pragma unroll
      for (int mi = 0; mi < S::MI; ++mi) {
#pragma unroll
        for (int r = 0; r < 4; ++r) m = fmaxf(m, acc[mi][ni][r]);
      }
      m = fmaxf(m, __shfl_xor(m, 16));
      m = fmaxf(m, __shfl_xor(m, 32));
      const float ref = safe(m);
      const int n = nbase + ni * 16;
      float s = 0.f;
      Power<T> out[S::MI][4];
#pragma unroll
      for (int mi = 0; mi < S::MI; ++mi) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float e = power(acc[mi][ni][r], ref);
          s += e;
          out[mi][r] = (Power<T>)(e * LIFT<T>);
        }
      }
      if constexpr (MODE == KEEP) {
        tile::store_columns<Power<T>, S::MI * 16>(
            out, stage + (ni & 1) * (S::MI * 256 * sizeof(T)),
            reinterpret_cast<Power<T>*>(grad) +
                (long)(n0 + wcol + ni * 16) * p.ldg + m0 + wrow,
            p.ldg, rows - (n0 + wcol + ni * 16), (int)p.ldg - (m0 + wrow), lane);
      }
      s += __shfl_xor(s, 16);
      s += __shfl_xor(s, 32);
      float z = zs[ni];
      if (p.pz) {
        z += __shfl_xor(z, 16);
        z += __shfl_xor(z, 32);
      }
      if (g == 0 && n < rows) {
        const long at = (long)n * p.bands + tm * S::WM + wave / S::WN;
        p.pmax[at] = m;
        p.psum[at] = s;
        if (p.pz) p.pz[at] = z;
      }
    }
  } else {
    float m[S::NI], k[S::NI], c[S::NI];
#pragma unroll
    for (int ni = 0; ni < S::NI; ++ni) {
      const int n = nbase + ni * 16;
      const bool in = n < rows;
      c[ni] = in ? p.coef[n] : 0.f;
      m[ni] = in ? p.rowm[n] : 0.f;
      k[ni] = in ? p.rowi[n] * c[ni] : 0.f;
    }
#pragma unroll
    for (int mi = 0; mi < S::MI; ++mi) {
#pragma unroll
      for (int ni = 0; ni < S::NI; ++ni) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          acc[mi][ni][r] = fmaf(power(acc[mi][ni][r], m[ni]), k[ni],
                                -p.share * c[ni]);
        }
      }
    }
#pragma unroll
    for (int ni = 0; ni < S::NI; ++ni) {
      if (t[ni] >= 0) {
        const float less = (1.f - p.eps) * c[ni];
#pragma unroll
        for (int q = 0; q < S::MI * 4; ++q) {
          acc[q >> 2][ni][q & 3] -=
              t[ni] == (q >> 2) * 16 + (q & 3) ? less : 0.f;
        }
      }
    }
    if (!whole) {
#pragma unroll
      for (int mi = 0; mi < S::MI; ++mi) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (vbase + mi * 16 + r >= p.vocab) {
#pragma unroll
            for (int ni = 0; ni < S::NI; ++ni) acc[mi][ni][r] = 0.f;
          }
        }
      }
    }
#pragma unroll
    for (int ni = 0; ni < S::NI; ++ni) {
      T out[S::MI][4];
#pragma unroll
      for (int mi = 0; mi < S::MI; ++mi) {
#pragma unroll
        for (int r = 0; r < 4; ++r) out[mi][r] = (T)acc[mi][ni][r];
      }
      tile::store_columns<T, S::MI * 16>(
          out, stage + (ni & 1) * (S::MI * 256 * sizeof(T)),
          grad + (long)(n0 + wcol + ni * 16) * p.ldg + m0 + wrow, p.ldg,
          rows - (n0 + wcol + ni * 16), (int)p.ldg - (m0 + wrow), lane);
    }
    if (p.pbias) {  // summed before the rounding
      __syncthreads();
      float* red = reinterpret_cast<float*>(smem);
#pragma unroll
      for (int mi = 0; mi < S::MI; ++mi) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float s = 0.f;
#pragma unroll
          for (int ni = 0; ni < S::NI; ++ni) {
            s += nbase + ni * 16 < rows ? acc[mi][ni][r] : 0.f;
          }
          s += __shfl_xor(s, 1);
          s += __shfl_xor(s, 2);
          s += __shfl_xor(s, 4);
          s += __shfl_xor(s, 8);
          if (i == 0) {
            red[(wave % S::WN) * S::BM + wrow + mi * 16 + g * 4 + r] = s;
          }
        }
      }
      __syncthreads();
      for (int q = threadIdx.x; q < S::BM; q += S::THREADS) {
        if (m0 + q >= p.vocab) continue;
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < S::WN; ++j) s += red[j * S::BM + q];
        p.pbias[(long)tn * p.all + p.v0 + m0 + q] = s;
      }
    }
  }
}

// One wave per row of the call: joins the bands.  rowm is the row's largest z
// and rowi the inverse of its sum, p = power(z, rowm) rowi.
__global__ __launch_bounds__(256) void join_kernel(
    const float* __restrict__ pmax, const float* __restrict__ psum,
    const float* __restrict__ pz, const float* __restrict__ ztgt,
    const int* __restrict__ pos, const int* __restrict__ tgt, long rows,
    int bands, float eps, float share, float* __restrict__ rowm,
    float* __restrict__ rowi, float* __restrict__ loss) {
  const int lane = threadIdx.x & 63;
  const long n = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (n >= rows) return;
  const int p = pos[n];
  if (p < 0) {
    if (lane == 0) loss[n] = 0.f;
    return;
  }
  const long at = (long)p * bands;
  constexpr int U = 8;  // bands of a lane in flight
  float m = -INFINITY, s = 0.f, z = 0.f;
  for (int base = lane; base < bands; base += 64 * U) {
    float a[U], b[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int k = base + 64 * j;
      a[j] = k < bands ? pmax[at + k] : -INFINITY;
      b[j] = k < bands ? psum[at + k] : 0.f;
      if (pz) z += k < bands ? pz[at + k] : 0.f;
    }
    float top = m;
#pragma unroll
    for (int j = 0; j < U; ++j) top = fmaxf(top, a[j]);
    s *= power(m, safe(top));
#pragma unroll
    for (int j = 0; j < U; ++j) {
      s = fmaf(b[j], power(a[j], safe(top)), s);
    }
    m = top;
  }
  const float top = safe(wave_max(m));
  s = wave_sum(s * power(m, top));
  z = wave_sum(z);
  if (lane == 0) {
    const bool bad = tgt[p] == BAD;
    rowm[p] = top;
    rowi[p] = bad ? NAN : 1.f / s;
    double v = (double)top + log((double)s) -
               (1.0 - (double)eps) * (double)ztgt[p];
    if (pz) v -= (double)share * (double)z;
    loss[n] = bad ? NAN : (float)v;
  }
}

// The sum of all losses (/ count for the mean), by one workgroup of any size,
// in a fixed order.
__device__ __forceinline__ void total_body(const float* loss, long rows,
                                           int count, bool mean,
                                           float* total) {
  __shared__ double part[16];
  double s = 0.0;
  for (long n = threadIdx.x; n < rows; n += blockDim.x) s += (double)loss[n];
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) s += __shfl_xor(s, k);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (unsigned k = 0; k < blockDim.x >> 6; ++k) t += part[k];
    *total = (float)(mean ? t / (double)count : t);
  }
}

__global__ __launch_bounds__(1024) void total_kernel(
    const float* __restrict__ loss, long rows, const int* __restrict__ count,
    int mean, float* __restrict__ total) {
  total_body(loss, rows, *count, mean, total);
}

// ------------------------------------------------------ factors and scales
// d(total)/d(loss) of a row is one (mean: 1 / count) times the upstream
// factor.  In 16 bits g is made with another factor, `lift`, and the products
// are scaled in fp32, for two reasons.  Where p is small, most of a row's g is
// its target's entry, -(1 - eps) factor: with factor = 1 / (1 - eps), times a
// power of two, that is -1 and rounds to itself, where one / count or 0.9 would
// be off by up to 2^-9 in every row alike (bf16, 2976 rows, eps 0.1: gradients
// off by 2.9e-3 of their norm instead of 1.9e-3).  And fp16 holds g to 6e-8
// only, so there the power of two is 2^14: |g| stays within 2^15, the type ends
// at 65504.
struct Factor {
  const float* scale;  // [1]: the inverse of the rows' own lift, or null
  const int* count;
  bool mean;
  float lift;  // 0: g is made with the factor itself

  __device__ __forceinline__ float one() const {
    return mean ? 1.f / (float)*count : 1.f;
  }
  __device__ __forceinline__ float lifted() const {
    return lift != 0.f ? lift : one();
  }
  __device__ __forceinline__ float inverse() const {
    if (scale) return scale[1];
    return lift != 0.f && *count > 0 ? one() / lift : 1.f;
  }
};

// ------------------------------------------------- g from the kept powers
// In place: g = c (power exp(band - row) / sum - eps / V), the target's entry
// anew from its z.  A workgroup takes `part` tokens, a lane one 16-byte chunk
// of each of them, and sums the bias gradient down the rows in passing; one
// more workgroup adds up the losses.  Bound by memory: 8 chunks are loaded
// before the first is used, the tokens' own factors are held by the lanes of a
// wave and read from there, and neighbouring workgroups take neighbouring
// columns (2976 kept rows of 9521 in bf16: 23 us, 5.0 TB/s, against 29 with
// one token after the other; 8192 of 30522: 197, 205 with the rows first).
// Down to 4 tokens a workgroup, 64 at most, where there would be fewer than 512
// workgroups otherwise; the parts of the bias gradient cost more from there on
// (700 x 33278: 20 us at 512, 28 at 2048).
template <class T>
__global__ __launch_bounds__(256) void probs_kernel(
    T* __restrict__ grad, long ldg, int vocab, int part, int columns,
    const int* __restrict__ tgt, const float* __restrict__ pmax, int bands,
    int band, const float* __restrict__ rowm, const float* __restrict__ rowi,
    const float* __restrict__ ztgt, const Factor factor, float eps,
    float share, float* __restrict__ pbias, const float* __restrict__ loss,
    long all, float* __restrict__ total) {
  constexpr int E = 16 / sizeof(T);
  const int rows = *factor.count;
  if (blockIdx.x == gridDim.x - 1) {
    total_body(loss, all, rows, factor.mean, total);
    return;
  }
  const int row = blockIdx.x / columns, column = blockIdx.x - row * columns;
  const int n0 = row * part;
  const int l = threadIdx.x & 63;
  const int lead = (column * 256 + (threadIdx.x - l)) * E;
  if (n0 >= rows || lead >= ldg) return;  // whole waves: lanes are read below
  const bool in = lead + l * E < ldg;
  const int v = in ? lead + l * E : (int)ldg - E;
  const int n1 = rows - n0 < part ? rows : n0 + part;
  const int mine = v / band;
  const float c = factor.lifted();
  // lane l of a wave: the factors of token n0 + l
  const int own = n0 + l < n1 ? n0 + l : n1 - 1;
  const float top = rowm[own], inv = rowi[own] * c;
  const int target = tgt[own];
  const float there =
      fmaf(power(ztgt[own], top), inv, -(share + (1.f - eps)) * c);
  const float times = inv * (1.f / LIFT<T>);
  const auto of = [](float x, int lane) {
    return __int_as_float(
        __builtin_amdgcn_readlane(__float_as_int(x), lane));
  };
  struct alignas(16) Powers {
    Power<T> v[E];
  };
  struct alignas(16) Chunk {
    T v[E];
  };
  constexpr int U = 8;  // tokens in flight
  float sum[E] = {};
  for (int n = n0; n < n1; n += U) {
    Powers t[U];
    float b[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int q = n + u < n1 ? n + u : n1 - 1;
      t[u] = *reinterpret_cast<const Powers*>(grad + (long)q * ldg + v);
      b[u] = pmax[(long)q * bands + mine];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (n + u >= n1) break;
      const int at = n + u - n0;
      // a band of nothing but -inf weighs nothing; taken for 0, it would be
      // past fp32 in a row whose largest z is below -88
      const float k = power(b[u], of(top, at)) * of(times, at);
      const int hit = __builtin_amdgcn_readlane(target, at) - v;
      const float h = of(there, at);
      float d[E];
#pragma unroll
      for (int j = 0; j < E; ++j) d[j] = fmaf((float)t[u].v[j], k, -share * c);
      if ((unsigned)hit < (unsigned)E) {
#pragma unroll
        for (int j = 0; j < E; ++j) d[j] = hit == j ? h : d[j];
      }
      if (v + E > vocab) {
#pragma unroll
        for (int j = 0; j < E; ++j) d[j] = v + j < vocab ? d[j] : 0.f;
      }
      Chunk g;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        sum[j] += d[j];
        g.v[j] = (T)d[j];
      }
      if (in) *reinterpret_cast<Chunk*>(grad + (long)(n + u) * ldg + v) = g;
    }
  }
  if (pbias && in) {
#pragma unroll
    for (int j = 0; j < E; ++j) {
      if (v + j < vocab) pbias[(long)row * vocab + v + j] = sum[j];
    }
  }
}

// ---------------------------------------------------------- row coefficients
// coef[i] = the factor of kept row i times scale[0], which brings the largest to
// `lift`; scale[1] is its inverse.
__global__ __launch_bounds__(1024) void coef_kernel(
    const float* __restrict__ up, int each, int mean,
    const int* __restrict__ idx, const int* __restrict__ tgt,
    const int* __restrict__ count, float lift, float* __restrict__ coef,
    float* __restrict__ scale) {
  __shared__ float part[16];
  __shared__ float shared_scale;
  const int rows = *count;
  const float one = each ? 1.f : (mean ? *up / (float)rows : *up);
  float top = 0.f;
  if (lift != 0.f) {
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
    // clamped: neither it nor its inverse leaves fp32
    const float s =
        m > 0.f ? fminf(fmaxf(lift / m, 0x1p-100f), 0x1p100f) : 1.f;
    shared_scale = s;
    scale[0] = s;
    scale[1] = 1.f / s;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows; i += 1024) {
    const float c = (each ? up[idx[i]] : one) * shared_scale;
    coef[i] = tgt[i] == BAD ? NAN : c;
  }
}

// ------------------------------------------- dx += g w and dw = g^T x
// Rows of dx's tiles are hidden units, columns tokens, k the piece's entries,
// cut into `splits` runs of `run` values that add to slabs of their own.  Rows
// of dw's tiles are hidden units, columns vocabulary entries, k tokens.
struct Dx {
  long ldw;
  int mt, splits, run, first;
  float* slabs;
  long slab;
  int blocks;
};

struct Dw {
  long ldx;
  int mt, nt, splits, run;
  void* out;
  float* slabs;
  long slab;
  int blocks;
};

template <class T, class S>
__device__ __forceinline__ void dx_body(const T* w, const T* grad, long ldg,
                                        int piece, int dim, int rows,
                                        const Dx& p, int block, char* smem) {
  const int nt = (rows + S::BN - 1) / S::BN;
  const int split = nt > 0 ? block / (p.mt * nt) : p.splits;
  if (split >= p.splits) return;
  int tm, tn;
  tile::pick(block - split * p.mt * nt, p.mt, nt, &tm, &tn);
  const int m0 = tm * S::BM, n0 = tn * S::BN;
  const int kbeg = split * p.run;
  const int kend = (int)ldg - kbeg < p.run ? (int)ldg : kbeg + p.run;
  f32x4 acc[S::MI][S::NI] = {};
  tile::product<T, true, false, S>(w, p.ldw, m0, dim, grad, ldg, n0, rows,
                                   kbeg, kend, piece, smem, acc, [] {});
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int i = lane & 15, g = lane >> 4;
  float* out = p.slabs + split * p.slab;
#pragma unroll
  for (int mi = 0; mi < S::MI; ++mi) {
    const int d = m0 + (wave / S::WN) * (S::MI * 16) + mi * 16 + g * 4;
    if (d >= dim) continue;  // dim is a multiple of 4
#pragma unroll
    for (int ni = 0; ni < S::NI; ++ni) {
      const int n = n0 + (wave % S::WN) * (S::NI * 16) + ni * 16 + i;
      if (n >= rows) continue;
      f32x4* at = reinterpret_cast<f32x4*>(out + (long)n * dim + d);
      *at = p.first ? acc[mi][ni] : *at + acc[mi][ni];
    }
  }
}

template <class T, class S>
__device__ __forceinline__ void dw_body(const T* x, const T* grad, long ldg,
                                        int piece, int dim, int ldim,
                                        int rows, const Factor& factor,
                                        const Dw& p, int block, char* smem) {
  const int split = block / (p.mt * p.nt);
  int tm, tn;
  tile::pick(block - split * p.mt * p.nt, p.mt, p.nt, &tm, &tn);
  const int m0 = tm * S::BM, n0 = tn * S::BN;
  const int kbeg = split * p.run;
  const int kend = rows - kbeg < p.run ? rows : kbeg + p.run;
  const float inv = factor.inverse();
  f32x4 acc[S::MI][S::NI] = {};
  tile::product<T, true, true, S>(x, p.ldx, m0, ldim, grad, ldg, n0,
                                  (int)ldg, kbeg, kend, kend, smem, acc,
                                  [] {});
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int i = lane & 15, g = lane >> 4;
  const int d0 = m0 + (wave / S::WN) * (S::MI * 16);
  T* out = (T*)p.out;
  char* stage = smem + wave * (2 * S::MI * 256 * sizeof(T));
#pragma unroll
  for (int ni = 0; ni < S::NI; ++ni) {
    const int v0 = n0 + (wave % S::WN) * (S::NI * 16) + ni * 16;
    if (!p.slabs) {
      T o[S::MI][4];
#pragma unroll
      for (int mi = 0; mi < S::MI; ++mi) {
#pragma unroll
        for (int r = 0; r < 4; ++r) o[mi][r] = (T)(acc[mi][ni][r] * inv);
      }
      char* to = stage + (ni & 1) * (S::MI * 256 * sizeof(T));
      T* at = out + (long)v0 * dim + d0;
      // as wide as the rows' alignment allows (13 x 16226 x 1982 in bf16, by
      // pairs: 38 us; values straight from the registers: 75)
      if (dim % (16 / (int)sizeof(T)) == 0) {
        tile::store_columns<T, S::MI * 16>(o, to, at, dim, piece - v0,
                                           dim - d0, lane);
      } else if (dim * sizeof(T) % 4 == 0) {
        tile::store_columns<T, S::MI * 16, int>(o, to, at, dim, piece - v0,
                                                dim - d0, lane);
      } else if constexpr (sizeof(T) == 2) {
        tile::store_columns<T, S::MI * 16, short>(o, to, at, dim, piece - v0,
                                                  dim - d0, lane);
      }
      continue;
    }
    const int v = v0 + i;
    if (v >= piece) continue;
#pragma unroll
    for (int mi = 0; mi < S::MI; ++mi) {
      const int d = d0 + mi * 16 + g * 4;
      if (d >= dim) continue;
      *reinterpret_cast<f32x4*>(p.slabs + split * p.slab + (long)v * ldim +
                                d) = acc[mi][ni];
    }
  }
}

// Both in one launch, the one with the longer runs first: alone, either leaves
// part of the card idle at its end (us, with the adding up after them: bf16,
// 700 x 33278 x 256: 43, 62 in two launches; 2976 kept of 3968 x 9521 x 512:
// 80, 104; fp32, 700 x 33278 x 256: 202, 217).
template <class T, class S>
__global__ __launch_bounds__(S::THREADS) void products_kernel(
    const T* __restrict__ w, const T* __restrict__ x,
    const T* __restrict__ grad, long ldg, int piece, int dim, int ldim,
    const Factor factor, const Dx dx, const Dw dw, int dw_first) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int rows = *factor.count;
  const int lead = dw_first ? dw.blocks : dx.blocks;
  const bool front = (int)blockIdx.x < lead;
  const int block = front ? blockIdx.x : blockIdx.x - lead;
  if (front == (dw_first != 0)) {
    dw_body<T, S>(x, grad, ldg, piece, dim, ldim, rows, factor, dw, block,
                  smem);
  } else {
    dx_body<T, S>(w, grad, ldg, piece, ldim, rows, dx, block, smem);
  }
}

// ------------------------------------------------------------- the endings
// Slabs of fp32 rows (ldim values, a multiple of 4) added into rows of `dim`
// values of T.  pos: which slab row a row takes, none (zeros) for -1.
struct Adding {
  const float* slabs;
  long slab, rows;
  int splits, ldim, dim;
  const int* pos;
  void* out;
  int blocks;
};

template <class T>
__device__ __forceinline__ void add_body(const Adding& a, float f,
                                         int block) {
  const int groups = (a.dim + 3) / 4;
  const long total = a.rows * groups;
  for (long k = (long)block * 256 + threadIdx.x; k < total;
       k += (long)a.blocks * 256) {
    const long n = k / groups;
    const int d = (int)(k - n * groups) * 4;
    const long p = a.pos ? a.pos[n] : n;
    f32x4 s = {};
    if (p >= 0) {
      const float* at = a.slabs + p * a.ldim + d;
#pragma unroll 8
      for (int j = 0; j < a.splits; ++j) {
        s += *reinterpret_cast<const f32x4*>(at + j * a.slab);
      }
    }
    T o[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = (T)(p >= 0 ? s[r] * f : 0.f);
    T* out = (T*)a.out + n * a.dim + d;
    if (d + 4 <= a.dim) {
      __builtin_memcpy(out, o, sizeof(o));
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (d + r < a.dim) out[r] = o[r];
      }
    }
  }
}

// db from its parts, of `part` tokens each: 64 entries a workgroup, 4 waves
// that take every fourth part
struct Bias {
  const float* parts;
  long vocab;
  int part;
  void* out;
  int blocks;
};

template <class T>
__device__ __forceinline__ void bias_body(const Bias& b, int rows, float f,
                                          int block) {
  __shared__ float sums[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long v = (long)block * 64 + lane;
  const int parts = (rows + b.part - 1) / b.part;
  float s = 0.f;
  if (v < b.vocab) {
#pragma unroll 8
    for (int k = wave; k < parts; k += 4) s += b.parts[(long)k * b.vocab + v];
  }
  sums[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && v < b.vocab) {
    ((T*)b.out)[v] =
        (T)((sums[0][lane] + sums[1][lane] + sums[2][lane] + sums[3][lane]) *
            f);
  }
}

// out *= up, where that changes anything; out is 16-byte aligned
struct Times {
  void* out;
  long n;
  int blocks;
};

template <class T>
__device__ __forceinline__ void times_body(const Times& t, float f,
                                           int block) {
  if (f == 1.f) return;
  constexpr int E = 16 / sizeof(T);
  struct alignas(16) Chunk {
    T v[E];
  };
  T* out = (T*)t.out;
  for (long k = (long)block * 256 + threadIdx.x; k * E < t.n;
       k += (long)t.blocks * 256) {
    if ((k + 1) * E <= t.n) {
      Chunk c = reinterpret_cast<Chunk*>(out)[k];
#pragma unroll
      for (int j = 0; j < E; ++j) c.v[j] = (T)((float)c.v[j] * f);
      reinterpret_cast<Chunk*>(out)[k] = c;
    } else {
      for (long j = k * E; j < t.n; ++j) out[j] = (T)((float)out[j] * f);
    }
  }
}

// The endings of one call in one launch, each with workgroups of its own.
template <class T>
__global__ __launch_bounds__(256) void end_kernel(
    const Adding dx, const Adding dw, const Bias db, const Times dw_times,
    const Factor factor, const float* __restrict__ up) {
  // no rows, no gradient, whatever the factor: 0 times infinity is none
  const bool any = *factor.count > 0;
  const float u = up && any ? *up : 1.f;
  const float f = any ? factor.inverse() * u : 0.f;
  int block = blockIdx.x;
  if (block < dx.blocks) return add_body<T>(dx, f, block);
  block -= dx.blocks;
  if (block < dw.blocks) return add_body<T>(dw, f, block);
  block -= dw.blocks;
  if (block < db.blocks) return bias_body<T>(db, *factor.count, f, block);
  times_body<T>(dw_times, u, block - db.blocks);
}

int blocks_for(long work) {
  return (int)std::min<long>(std::max<long>((work + 255) / 256, 1), 8192);
}

int ceil_div(long a, long b) { return (int)((a + b - 1) / b); }

using Wide = Shape<256, 256, 2, 4>;
using Mid = Shape<128, 128, 2, 4>;
using Small = Shape<128, 64, 2, 2>;
using Deep = Shape<64, 64, 2, 2, 3>;
using Thin = Shape<64, 32, 2, 2, 4>;

// Calls f with a value of the tile's shape; those that a type never takes are
// not built (SMALL: whether 16-bit types take that one).
template <class T, bool SMALL, class F>
void by_shape(Tile t, F f) {
  constexpr bool HALF = sizeof(T) == 2;
  if constexpr (HALF) {
    if (t == Tile::wide) return f(Wide());
    if (t == Tile::mid) return f(Mid());
  }
  if constexpr (SMALL || !HALF) {
    if (t == Tile::small) return f(Small());
  }
  if (t == Tile::deep) return f(Deep());
  f(Thin());
}

// Allows a kernel its LDS, once on each device.
template <auto KERNEL>
void with_lds(int bytes) {
  static std::atomic<uint64_t> done{0};
  int device = 0;
  check(hipGetDevice(&device));
  const uint64_t bit = 1ull << (device & 63);
  if (done.load(std::memory_order_relaxed) & bit) return;
  check(hipFuncSetAttribute(reinterpret_cast<const void*>(KERNEL),
                            hipFuncAttributeMaxDynamicSharedMemorySize,
                            bytes));
  done.fetch_or(bit, std::memory_order_relaxed);
}

// what g's factor is brought to, see Factor; 0 leaves it
template <class T>
float lift(float eps) {
  if (sizeof(T) == 4) return 0.f;
  const float top = std::is_same_v<T, _Float16> ? 0x1p14f : 1.f;
  return eps <= 0.5f ? top / (1.f - eps) : top;
}

template <class T>
struct Run {
  template <class S, int MODE>
  static void logits(const Operands& o, Logits p, T* grad, hipStream_t s) {
    p.ldw = o.ldw;
    p.ldx = o.ldx;
    p.mt = ceil_div(p.vocab, S::BM);
    const int nt = ceil_div(o.rows, S::BN);
    p.count = o.count;
    p.tgt = o.tgt;
    with_lds<logits_kernel<T, S, MODE>>(S::LDS);
    logits_kernel<T, S, MODE><<<p.mt * nt, S::THREADS, S::LDS, s>>>(
        (const T*)o.w, (const T*)o.x, (const T*)o.bias, grad, p);
    check(hipGetLastError());
  }

  static void forward(const Operands& o, const Sums& f, T* grad,
                      hipStream_t s) {
    Logits p{};
    p.vocab = (int)o.vocab;
    p.pmax = f.pmax;
    p.psum = f.psum;
    p.pz = o.eps != 0.f ? f.pz : nullptr;
    p.ztgt = f.ztgt;
    p.bands = o.plan.bands;
    p.ldg = padded(o.vocab);
    by_shape<T, true>(o.plan.logits, [&](auto shape) {
      using S = decltype(shape);
      if (grad) {
        logits<S, KEEP>(o, p, grad, s);
      } else {
        logits<S, SUMS>(o, p, nullptr, s);
      }
    });
    join_kernel<<<ceil_div(o.rows, 4), 256, 0, s>>>(
        f.pmax, f.psum, p.pz, f.ztgt, o.pos, o.tgt, o.rows, p.bands, o.eps,
        o.eps / (float)o.vocab, f.rowm, f.rowi, f.loss);
    check(hipGetLastError());
  }

  static Factor factor(const Operands& o, const Grads& b) {
    return Factor{b.scale, o.count, b.mean, lift<T>(o.eps)};
  }

  static void probs(const Operands& o, const Sums& f, const Grads& b,
                    hipStream_t s) {
    const long ldg = padded(o.vocab);
    const int columns = ceil_div(ldg * sizeof(T) / 16, 256);
    probs_kernel<T><<<ceil_div(o.rows, o.plan.part) * columns + 1, 256, 0,
                      s>>>(
        (T*)b.grad, ldg, (int)o.vocab, o.plan.part, columns, o.tgt, f.pmax,
        o.plan.bands, o.plan.band, f.rowm, f.rowi, f.ztgt, factor(o, b),
        o.eps, o.eps / (float)o.vocab, b.pbias, f.loss, o.rows, f.total);
    check(hipGetLastError());
  }

  static void again(const Operands& o, const Sums& f, const Grads& b,
                    long v0, int piece, hipStream_t s) {
    Logits p{};
    p.v0 = (int)v0;
    p.vocab = piece;
    p.ldg = padded(piece);
    p.rowm = f.rowm;
    p.rowi = f.rowi;
    p.coef = b.coef;
    p.eps = o.eps;
    p.share = o.eps / (float)o.vocab;
    p.pbias = b.pbias;
    p.all = o.vocab;
    by_shape<T, true>(o.plan.logits, [&](auto shape) {
      logits<decltype(shape), AGAIN>(o, p, (T*)b.grad, s);
    });
  }

  template <class S>
  static void products_as(const Operands& o, const Grads& b, long v0,
                          int piece, hipStream_t s) {
    const int md = ceil_div(o.ldx, S::BM);
    Dx dx{};
    Dw dw{};
    if (b.dx_slabs) {
      dx.ldw = o.ldw;
      dx.mt = md;
      dx.splits = o.plan.dx_splits;
      dx.run = ceil_div(ceil_div(padded(piece), dx.splits), 64) * 64;
      dx.first = v0 == 0;
      dx.slabs = b.dx_slabs;
      dx.slab = o.rows * o.ldx;
      dx.blocks = md * ceil_div(o.rows, S::BN) * dx.splits;
    }
    if (b.dw || b.dw_slabs) {
      dw.ldx = o.ldx;
      dw.mt = md;
      dw.nt = ceil_div(piece, S::BN);
      dw.splits = o.plan.dw_splits;
      dw.run = ceil_div(ceil_div(o.rows, dw.splits), 64) * 64;
      dw.out = (T*)b.dw + v0 * o.dim;
      dw.slabs = b.dw_slabs;
      dw.slab = (long)piece * o.ldx;
      dw.blocks = md * dw.nt * dw.splits;
    }
    if (dx.blocks + dw.blocks == 0) return;
    with_lds<products_kernel<T, S>>(S::LDS);
    products_kernel<T, S><<<dx.blocks + dw.blocks, S::THREADS, S::LDS, s>>>(
        (const T*)o.w + v0 * o.ldw, (const T*)o.x, (const T*)b.grad,
        padded(piece), piece, o.dim, o.ldx, factor(o, b), dx, dw,
        dw.run > dx.run);
    check(hipGetLastError());
  }

  static void products(const Operands& o, const Grads& b, long v0, int piece,
                       hipStream_t s) {
    by_shape<T, false>(o.plan.grads, [&](auto shape) {
      products_as<decltype(shape)>(o, b, v0, piece, s);
    });
  }

  // What is left of rows [v0, v0 + piece) of dw, and of dx and db where they
  // are given, times up (null: 1).
  static void end(const Operands& o, const Grads& b, long v0, int piece,
                  bool rest, const float* up, hipStream_t s) {
    const int groups = (o.dim + 3) / 4;
    Adding dx{}, dw{};
    Bias db{};
    Times times{};
    if (rest && b.dx) {
      dx = Adding{b.dx_slabs, o.rows * o.ldx, o.rows, o.plan.dx_splits, o.ldx,
                  o.dim, o.pos, b.dx, blocks_for(o.rows * groups)};
    }
    if (b.dw && b.dw_slabs) {
      dw = Adding{b.dw_slabs, (long)piece * o.ldx, piece, o.plan.dw_splits,
                  o.ldx, o.dim, nullptr, (T*)b.dw + v0 * o.dim,
                  blocks_for((long)piece * groups)};
    } else if (b.dw && up) {
      times.out = b.dw;
      times.n = o.vocab * o.dim;
      times.blocks = std::min(blocks_for(times.n / 8), 2048);
    }
    if (rest && b.db) {
      db = Bias{b.pbias, o.vocab, o.plan.part, b.db, ceil_div(o.vocab, 64)};
    }
    const int blocks = dx.blocks + dw.blocks + db.blocks + times.blocks;
    if (blocks == 0) return;
    end_kernel<T><<<blocks, 256, 0, s>>>(dx, dw, db, times, factor(o, b), up);
    check(hipGetLastError());
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

constexpr int EDGE_M[] = {256, 128, 128, 64, 64};
constexpr int EDGE_N[] = {256, 128, 64, 64, 32};
constexpr int BAND[] = {128, 64, 64, 32, 32};
long tiles(Tile t, long m, long n) {
  return (long)ceil_div(m, EDGE_M[(int)t]) * ceil_div(n, EDGE_N[(int)t]);
}

// -------------------------------------------------------- choosing the tiles
// A launch's time by a simple count.  A CU has as many places as workgroups fit
// into its LDS; a workgroup takes `start` us and per slice of k `alone` us, or
// `shared` us for each of those that share its CU if that is more.  The figures
// are fitted to measured times.
struct Speed {
  float shared, alone, start;
  int places;

  float slice(long workgroups) const {
    const float share =
        std::min(std::max(workgroups / 256.f, 1.f), (float)places);
    return std::max(alone, shared * share);
  }
  long all_places(long workgroups) const {
    return workgroups > 256 ? 256 * places : 256;
  }
};
constexpr float SLAB = 0.3e-6f;  // us a byte of fp32 that is written and read

// Logits: 242 times of 48 shapes, with and without the powers.  What the count
// takes is 0.4% slower than the best of each on the mean, at worst 5% (fp32:
// 0.1%; a rule on the number of tiles, which took deep ones for 70 x 2246 x
// 2080 in fp32, 37 us against 22 with thin ones, was 13% slower there).
// wide: twice the work per byte that goes through LDS, but one workgroup fills
//   a CU (bf16, 16384 x 8192 x 768: 217, mid 251; 5081 x 6852 x 32: 31, mid 27).
// mid: a short k, some hundred rows (37215 x 88 x 416: 12.8, wide 18.6, small
//   13.6).
// small: fp32 products are 16 times slower for the same loads, so more
//   workgroups to a CU lose nothing (9521 x 4096 x 1024: 590, deep 611); in 16
//   bits up to 64 rows (33278 x 35 x 256: 7.6, wide 14.2, mid 9.0).
// deep, thin: few tiles, or few rows (fp32, 30522 x 8 x 768: thin 18.5, small
//   29; bf16, 2636 x 196 x 288: deep 5.8, mid 8.0).
constexpr Speed HALF_LOGITS[] = {{1.13f, 1.19f, 9.3f, 1},
                                 {0.48f, 0.57f, 4.4f, 2},
                                 {0.36f, 0.37f, 4.1f, 3},
                                 {0.23f, 0.25f, 4.1f, 3},
                                 {0.09f, 0.2f, 3.4f, 3}};
constexpr Speed FULL_LOGITS[] = {{},
                                 {},
                                 {1.0f, 0.91f, 5.1f, 3},
                                 {0.55f, 0.52f, 4.3f, 3},
                                 {0.24f, 0.285f, 3.7f, 3}};

Tile logits_tile(long vocab, long rows, long k, int size) {
  const float slices = (float)ceil_div(k * size, 128);
  Tile taken = Tile::thin;
  float best = INFINITY;
  for (int t = 0; t < 5; ++t) {
    const Speed& speed = (size == 2 ? HALF_LOGITS : FULL_LOGITS)[t];
    if (speed.places == 0) continue;
    const long all = tiles((Tile)t, vocab, rows);
    const float one = speed.start + slices * speed.slice(all);
    const float rounds = (float)all / speed.all_places(all);
    // a last round that is filled in part takes half a round and half its part
    const float whole = std::floor(rounds), part = rounds - whole;
    const float cost =
        one * (whole + (whole == 0.f ? 1.f
                        : part > 0.f ? 0.5f + 0.5f * part : 0.f)) +
        SLAB * 8 * rows * (float)(vocab / BAND[t]);
    if (cost < best) {
      best = cost;
      taken = (Tile)t;
    }
  }
  return taken;
}

// ------------------------------------------------ the tiles of the gradients
// dw has the vocabulary's many tiles and a k of the rows; dx has few tiles and
// a k of the vocabulary, so that is cut up into runs, each of which writes
// fp32 partial sums that are read once more; so is the k of dw where its tiles
// do not fill the card.  The workgroups of both products, the longer ones
// first, go to the first free place.  1319 measured times of 30 shapes (1 to
// 8192 rows, 600 to 100000 entries, 32 to 2048 values): what the count takes is
// 2% slower than the best of each on the mean, at worst 15% (102 x 11354 x 32:
// 11.2 us, 9.7); on 8 others, of few rows and large weights, 4% on the mean, at
// worst 7%.  A rule for each product by itself, that filled the card with it,
// was 25% slower on the mean.
constexpr Speed HALF_SPEED[] = {{1.1f, 0.8f, 8.3f, 1},
                                {0.44f, 0.74f, 3.5f, 2},
                                {},
                                {0.194f, 0.28f, 3.8f, 3},
                                {0.14f, 0.2f, 3.8f, 3}};
constexpr Speed FULL_SPEED[] = {{},
                                {},
                                {0.78f, 0.97f, 4.8f, 3},
                                {0.343f, 0.5f, 4.6f, 3},
                                {0.216f, 0.33f, 3.0f, 3}};
constexpr int RUNS[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64};

// The end of n1 jobs of length a and then n2 of length b <= a on `places`.
float ending(long n1, float a, long n2, float b, long places) {
  const long late = n1 % places;  // places that are free one job later
  const float lo = n1 / places * a, hi = late ? lo + a : lo;
  if (n2 == 0) return hi;
  const long behind = late ? (long)std::ceil(a / b) : 0;
  long k = (n2 + places - late - 1) / (places - late);
  if (k > behind) k = (n2 + late * behind + places - 1) / places;
  float end = lo + k * b;
  const long m = k - behind;  // does it end with the late ones' last job?
  if (late && m >= 0 &&
      (places - late) * (m + (long)(a / b)) + late * m >= n2) {
    end = hi + m * b;
  }
  return std::max(end, hi);
}

void plan_grads(Plan* p, long rows, long ldim, int size) {
  const long unit = 128 / size, piece = p->piece;
  float best = INFINITY;
  for (int t = 0; t < 5; ++t) {
    const Speed& speed = (size == 2 ? HALF_SPEED : FULL_SPEED)[t];
    if (speed.places == 0) continue;
    const long nx = tiles((Tile)t, ldim, rows), nw = tiles((Tile)t, ldim, piece);
    const long most =
        std::max<long>(1, std::min<long>({256 / nw, rows / 512, 16}));
    for (long cuts = 1;; cuts = most) {
      const float b = (float)ceil_div(ceil_div(rows, cuts), unit);
      for (int runs : RUNS) {
        if (runs > 1 && runs * 128 > piece) break;
        const float a = (float)ceil_div(ceil_div(piece, runs), unit);
        const long all = nx * runs + nw * cuts;
        const float slice = speed.slice(all);
        const long places = speed.all_places(all);
        const float ta = speed.start + a * slice, tb = speed.start + b * slice;
        const float cost =
            (a >= b ? ending(nx * runs, ta, nw * cuts, tb, places)
                    : ending(nw * cuts, tb, nx * runs, ta, places)) +
            SLAB * 4 * ldim * ((float)runs * rows +
                               (cuts > 1 ? (float)cuts * piece : 0.f));
        if (cost < best) {
          best = cost;
          p->grads = (Tile)t;
          p->dx_splits = runs;
          p->dw_splits = (int)cuts;
        }
      }
      if (cuts == most) break;
    }
  }
}

Plan make_plan(long rows, long vocab, int ldim, int size, bool keep) {
  Plan p;
  p.logits = logits_tile(vocab, rows, ldim, size);
  p.band = BAND[(int)p.logits];
  const int edge_m = EDGE_M[(int)p.logits], edge_n = EDGE_N[(int)p.logits];
  p.bands = ceil_div(vocab, edge_m) * (edge_m / p.band);
  // a piece of the vocabulary: 256 MB of g at most, which the card's last
  // cache then holds between the three products; offsets within a tile of g
  // stay below 2^31 for rows of up to a million entries
  const long most = std::min<long>(
      std::max<long>((256l << 20) / (rows * size), edge_m), 1l << 20);
  p.piece = keep ? vocab : std::min(vocab, most / edge_m * edge_m);
  p.part = edge_n;
  if (keep) {
    const long columns = ceil_div(vocab * size, 4096);
    p.part = 64;
    while (p.part > 4 && columns * ceil_div(rows, p.part) < 512) p.part /= 2;
  }
  p.parts = ceil_div(rows, p.part);
  plan_grads(&p, rows, ldim, size);
  return p;
}

}  // namespace

long padded(long n) { return (n + 7) / 8 * 8; }

// The last sizes' plan is kept: the steps of a loop have the same, and the
// count over tiles and runs takes a launch's time.
Plan plan(long rows, long vocab, int ldim, int size, bool keep) {
  struct Last {
    long rows = -1, vocab = 0;
    int ldim = 0, size = 0;
    bool keep = false;
    Plan plan;
  };
  thread_local Last last;
  if (last.rows != rows || last.vocab != vocab || last.ldim != ldim ||
      last.size != size || last.keep != keep) {
    last.plan = make_plan(rows, vocab, ldim, size, keep);
    last.rows = rows;
    last.vocab = vocab;
    last.ldim = ldim;
    last.size = size;
    last.keep = keep;
  }
  return last.plan;
}

long work_items(const Plan& p, long rows, long vocab, int ldim, int size,
                bool keep) {
  static_assert(Wide::THREADS == 512 && Mid::THREADS == 512 &&
                    Small::THREADS == 256 && Deep::THREADS == 256 &&
                    Thin::THREADS == 256, "as below");
  const auto threads = [](Tile t) {
    return t == Tile::wide || t == Tile::mid ? 512l : 256l;
  };
  const auto blocks = [](long a, long b) { return (a + b - 1) / b; };
  const long logits = tiles(p.logits, vocab, rows) * threads(p.logits);
  const long grads = (tiles(p.grads, ldim, rows) * p.dx_splits +
                      tiles(p.grads, ldim, p.piece) * p.dw_splits) *
                     threads(p.grads);
  const long join = blocks(rows, 4) * 256;
  const long probs =
      keep ? (blocks(rows, p.part) * blocks(padded(vocab) * size, 4096) + 1) *
                 256
           : 0;
  const long end = (3 * 8192 + blocks(vocab, 64)) * 256;
  return std::max({logits, grads, join, probs, end});
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

template <class T>
Loads loads_of(const void* in, long ld, long step, int cols, int ldo) {
  const auto aligned = [&](long n) {
    return step == 1 && (uintptr_t)in % n == 0 && ld * sizeof(T) % n == 0;
  };
  return ldo == cols && aligned(16) ? WIDE : aligned(4) ? PAIRS : SINGLE;
}

void pack(Type t, const void* in, long ld, long step, long rows, int cols,
          const int* idx, const int* count, void* out, int ldo,
          hipStream_t s) {
  by_type(t, [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    int lanes = 0;
    while (lanes < 6 && 16 << lanes < ldo * (int)sizeof(T)) ++lanes;
    pack_kernel<T><<<blocks_for(rows << lanes), 256, 0, s>>>(
        (const T*)in, ld, step, rows, cols, idx, count, (T*)out, ldo,
        loads_of<T>(in, ld, step, cols, ldo), lanes);
    check(hipGetLastError());
  });
}

void prepare(Type t, const void* target, bool wide_ints, long rows,
             long ignore, long vocab, int* pos, int* idx, int* tgt,
             int* count, const void* in, long ld, long step, int cols,
             void* out, int ldo, hipStream_t s) {
  if (rows > PREP_MOST) {
    scan(target, wide_ints, rows, ignore, vocab, pos, idx, tgt, count, s);
    pack(t, in, ld, step, rows, cols, idx, count, out, ldo, s);
    return;
  }
  by_type(t, [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    auto launch = [&](auto* targets) {
      // few rows: more workgroups (60 rows of 4096 in bf16: 4.8 us by
      // single rows, 8 by 4)
      const int prep = rows <= 512 ? 1 : rows <= 4096 ? 4 : PREP;
      prepare_kernel<<<ceil_div(rows, prep), 256, 0, s>>>(
          targets, rows, ignore, vocab, pos, idx, tgt, count, (const T*)in,
          ld, step, cols, (T*)out, ldo,
          (int)loads_of<T>(in, ld, step, cols, ldo), prep);
      check(hipGetLastError());
    };
    if (wide_ints) {
      launch((const long*)target);
    } else {
      launch((const int*)target);
    }
  });
}

void forward(Type t, const Operands& o, const Sums& f, void* grad,
             hipStream_t s) {
  by_type(t, [&](auto* q) {
    using T = std::remove_pointer_t<decltype(q)>;
    Run<T>::forward(o, f, (T*)grad, s);
  });
}

void total(const float* loss, long rows, const int* count, bool mean,
           float* out, hipStream_t s) {
  total_kernel<<<1, 1024, 0, s>>>(loss, rows, count, mean, out);
  check(hipGetLastError());
}

void coefficients(Type t, const Operands& o, const float* up, bool each,
                  const Grads& b, hipStream_t s) {
  by_type(t, [&](auto* q) {
    using T = std::remove_pointer_t<decltype(q)>;
    coef_kernel<<<1, 1024, 0, s>>>(up, each, b.mean, o.idx, o.tgt, o.count,
                                   lift<T>(o.eps), b.coef, b.scale);
    check(hipGetLastError());
  });
}

void gradients_kept(Type t, const Operands& o, const Sums& f, const Grads& b,
                    hipStream_t s) {
  by_type(t, [&](auto* q) {
    using T = std::remove_pointer_t<decltype(q)>;
    Run<T>::probs(o, f, b, s);
    Run<T>::products(o, b, 0, (int)o.vocab, s);
  });
}

void finish_kept(Type t, const Operands& o, const Grads& b, const float* up,
                 hipStream_t s) {
  by_type(t, [&](auto* q) {
    using T = std::remove_pointer_t<decltype(q)>;
    Run<T>::end(o, b, 0, (int)o.vocab, true, up, s);
  });
}

void gradients_again(Type t, const Operands& o, const Sums& f, const Grads& b,
                     hipStream_t s) {
  by_type(t, [&](auto* q) {
    using T = std::remove_pointer_t<decltype(q)>;
    for (long v0 = 0; v0 < o.vocab; v0 += o.plan.piece) {
      const int piece = (int)std::min(o.plan.piece, o.vocab - v0);
      Run<T>::again(o, f, b, v0, piece, s);
      Run<T>::products(o, b, v0, piece, s);
      Run<T>::end(o, b, v0, piece, v0 + piece == o.vocab, nullptr, s);
    }
  });
}

}  // namespace vocab_loss
