// Launchers of the vocabulary-loss kernels (vocab_loss.hip), free of torch so
// that the kernels build in seconds.  All pointers are device memory.
#pragma once

#include <hip/hip_runtime.h>

#include <stdexcept>
#include <string>

namespace vocab_loss {

enum class Type { bf16, fp16, fp32 };

constexpr int BAD = -(1 << 30);  // a kept row whose target is no entry

inline void check(hipError_t e) {
  if (e != hipSuccess) {
    throw std::runtime_error(std::string("HIP error: ") +
                             hipGetErrorString(e));
  }
}

// 256 x 256, 128 x 128, 128 x 64; 64 x 64 and 64 x 32 with more slices of k on
// their way
enum class Tile { wide, mid, small, deep, thin };

// How a call of given sizes is cut up.
struct Plan {
  Tile logits, grads;
  int band, bands;        // entries of a band, bands of a row
  long piece;             // entries of the vocabulary at a time
  int part, parts;        // tokens of a part of the bias gradient's sum
  int dx_splits, dw_splits;
};

// keep: the whole vocabulary's powers are kept for the gradients
Plan plan(long rows, long vocab, int ldim, int size, bool keep);
// Work items of a plan's largest launch.  The runtime launches fewer than 2^32.
long work_items(const Plan& p, long rows, long vocab, int ldim, int size,
                bool keep);

long padded(long n);  // to whole 16-byte chunks of every type

struct Operands {
  Plan plan;
  const void *w, *x, *bias;
  long ldw, rows, vocab;
  int ldx;  // packed x: kept rows by ldx values, zeros past the hidden size
  int dim;
  float eps;
  const int *pos, *idx, *tgt, *count;
};

struct Sums {
  float *pmax, *psum, *pz;             // [row][band]
  float *rowm, *rowi, *ztgt, *loss;    // [row]
  float* total;
};

struct Grads {
  float *coef, *scale, *pbias, *dx_slabs, *dw_slabs;
  void *grad, *dx, *dw, *db;
  bool mean;
};

// The kept rows of a call: numbers them (pos, idx, tgt, count) and packs their
// hidden states into rows of ldo values.
void prepare(Type t, const void* target, bool wide_ints, long rows,
             long ignore, long vocab, int* pos, int* idx, int* tgt,
             int* count, const void* in, long ld, long step, int cols,
             void* out, int ldo, hipStream_t s);
// The same of rows that are numbered already, or of all rows (idx null).
void pack(Type t, const void* in, long ld, long step, long rows, int cols,
          const int* idx, const int* count, void* out, int ldo,
          hipStream_t s);
// grad: where the powers go, or null
void forward(Type t, const Operands& o, const Sums& f, void* grad,
             hipStream_t s);
void total(const float* loss, long rows, const int* count, bool mean,
           float* out, hipStream_t s);
// up: one value, or one for each row (`each`)
void coefficients(Type t, const Operands& o, const float* up, bool each,
                  const Grads& b, hipStream_t s);
// these also write f.total
void gradients_kept(Type t, const Operands& o, const Sums& f, const Grads& b,
                    hipStream_t s);
void finish_kept(Type t, const Operands& o, const Grads& b, const float* up,
                 hipStream_t s);
void gradients_again(Type t, const Operands& o, const Sums& f, const Grads& b,
                     hipStream_t s);

}  // namespace vocab_loss
