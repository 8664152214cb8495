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

// How a call of given sizes is cut up.
struct Plan {
  bool wide;
  int edge, tiles, row_tiles, dx_splits, dw_splits;
  long piece;
};

Plan plan(long rows, long vocab, int ldim, int size);

struct Forward {
  Plan plan;
  const void *w, *x, *bias;
  long ldw, rows, vocab;
  int ldx;  // packed x: kept rows by ldx values, zeros past the hidden size
  float eps;
  const int *pos, *tgt, *count;
  float *pmax, *psum, *pz, *ztgt, *lse, *loss;
};

struct Backward {
  Plan plan;
  const void *w, *x, *bias;
  long ldw, rows, vocab, piece;
  int ldx, dim;
  float eps;
  const int *pos, *idx, *tgt, *count;
  const float* lse;
  const float* up;  // upstream gradient: one value, or one for each row
  bool each, mean;
  int dx_splits, dw_splits;
  float *coef, *scale, *pbias, *dx_slabs, *dw_slabs;
  void *grad, *dx, *dw, *db;
};

void scan(const void* target, bool wide_ints, long rows, long ignore,
          long vocab, int* pos, int* idx, int* tgt, int* count,
          hipStream_t s);
void pack(Type t, const void* in, long ld, long step, long rows, int cols,
          const int* idx, const int* count, void* out, int ldo,
          hipStream_t s);
void forward(Type t, const Forward& f, hipStream_t s);
void total(const float* loss, long rows, const int* count, bool mean,
           float* out, hipStream_t s);
void backward(Type t, const Backward& b, hipStream_t s);

}  // namespace vocab_loss
