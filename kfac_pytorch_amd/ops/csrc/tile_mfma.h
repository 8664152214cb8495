// The matrix-product loop that the vocabulary-loss kernels share.
//
// C[m, n] = sum_k A(m, k) B(n, k), fp32 accumulation, one BM x BN tile of C
// per workgroup.  An operand lies in memory either k-inner (row m, k
// contiguous) or k-outer (row k, m contiguous).  Both kinds are staged by
// 16-byte loads that go from memory straight to LDS, 128 bytes of k for each
// of the tile's rows, in two buffers: the loads of the next slice of k are in
// flight while the matrix cores work on this one.
//
// Loads straight to LDS write lane i's 16 bytes at base + 16 i, so a layout
// without bank conflicts is made by choosing which chunk each lane fetches:
//   k-inner: row r keeps its 16-byte chunk c at slot c ^ (r & 7); the 16 rows
//     of a fragment's chunk then fall on all bank groups.
//   k-outer, 16 bits: fragments are read by the transposing LDS read, whose 64
//     lanes touch 32 bytes of each of 16 k-rows; the 32-byte column is xored
//     with the 4 bits of k that tell those 16 rows apart.
//   k-outer, 32 bits: fragments are read word by word, 64 bytes of each of 4
//     k-rows; the 64-byte column is xored with the 2 bits of k.
//
// Rows past the end of an operand, and k past its end, are turned into
// out-of-range buffer offsets, for which the hardware returns zeros.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace tile {

using f32x4 = __attribute__((ext_vector_type(4))) float;
using s16x4 = __attribute__((ext_vector_type(4))) short;
using s16x8 = __attribute__((ext_vector_type(8))) short;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;
using lds_void = __attribute__((address_space(3))) void;
using lds_s16x4 = __attribute__((address_space(3))) s16x4;

constexpr uint32_t OUT_OF_RANGE = 0x7ffffff0u;
constexpr long MAX_RECORDS = 0x7fffff00l;

// A raw buffer of `bytes` bytes from p on.
using Rsrc = __attribute__((ext_vector_type(4))) int;
__device__ __forceinline__ Rsrc make_rsrc(const void* p, long bytes) {
  const long n = bytes < 0 ? 0 : (bytes > MAX_RECORDS ? MAX_RECORDS : bytes);
  const uint64_t at = reinterpret_cast<uint64_t>(p);
  return Rsrc{(int)(uint32_t)at, (int)(uint32_t)(at >> 32) & 0xffff, (int)n,
              0x00020000};
}

// Starts a load of 16 bytes a lane from buffer r at offset off + uniform,
// straight to LDS at `to` + 16 * lane.  Written as assembly because the
// compiler takes the builtin's write to LDS for an alias of every later LDS
// read and waits for it there; what orders the two here are the explicit wait
// and the barrier in product().  It has no register to return.
__device__ __forceinline__ void load_to_lds(Rsrc r, char* to, uint32_t off,
                                            uint32_t uniform) {
  const uint32_t at = (uint32_t)(uintptr_t)(lds_void*)to;
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %1, %2, %3 offen lds"
      :
      : "s"(at), "v"(off), "s"(r), "s"(uniform)
      : "m0", "memory");
}

// All LDS reads of this wave have arrived and all but its last LATER loads to
// LDS, and the other waves are as far.  (vmcnt counts loads in the order they
// were started; other accesses in flight only make the wait longer.)
template <int LATER>
__device__ __forceinline__ void arrive() {
  static_assert(LATER < 64, "six bits of count");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt((LATER & 15) | 7 << 4 | (LATER >> 4) << 14);
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
  __builtin_amdgcn_sched_barrier(0);
}

// one 16-byte fragment piece: 8 values of 16 bits, or 4 of 32
union Frag {
  s16x8 h;
  f32x4 f;
  s16x4 q[2];
  float w[4];
};

template <class T>
__device__ __forceinline__ f32x4 mma(const Frag& a, const Frag& b, f32x4 c);

template <>
__device__ __forceinline__ f32x4 mma<__bf16>(const Frag& a, const Frag& b,
                                             f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(
      __builtin_bit_cast(bf16x8, a.h), __builtin_bit_cast(bf16x8, b.h), c, 0,
      0, 0);
}
template <>
__device__ __forceinline__ f32x4 mma<_Float16>(const Frag& a, const Frag& b,
                                               f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(
      __builtin_bit_cast(f16x8, a.h), __builtin_bit_cast(f16x8, b.h), c, 0, 0,
      0);
}
// lane group l >> 4 holds 4 consecutive k of its row; the instruction takes
// one k of each group, and any pairing of k will do that both operands share
template <>
__device__ __forceinline__ f32x4 mma<float>(const Frag& a, const Frag& b,
                                            f32x4 c) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.f[j], b.f[j], c, 0, 0, 0);
  }
  return c;
}

template <class T>
constexpr int MMAS = sizeof(T) == 2 ? 1 : 4;  // instructions of one mma()

// Asks the scheduler to start with a matrix instruction (its operands have
// been read long before) and to put the LDS reads singly between the next
// ones, so that the last has arrived when the block ends.
template <int MATRIX, int READS>
__device__ __forceinline__ void spread() {
  constexpr int EACH = MATRIX / 4 * 3 / READS > 0 ? MATRIX / 4 * 3 / READS : 1;
#pragma unroll
  for (int i = 0; i < READS; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);  // matrix
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);     // LDS read
  }
  __builtin_amdgcn_sched_group_barrier(0x008, MATRIX, 0);
}

// A tile shape: BM x BN of C by WM x WN waves, with ST slices of k in LDS or
// on their way there.
template <int BM_, int BN_, int WM_, int WN_, int ST_ = 2>
struct Shape {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, ST = ST_;
  static constexpr int NW = WM * WN, THREADS = NW * 64;
  static constexpr int MI = BM / WM / 16, NI = BN / WN / 16;
  static constexpr int SLICE = (BM + BN) * 128, LDS = ST * SLICE;
};

// One operand of a tile: R rows (of C's rows or columns).
template <class T, bool KOUTER, int R, int NW>
struct Operand {
  static constexpr int SZ = sizeof(T);
  static constexpr int E = 16 / SZ;       // values in a chunk
  static constexpr int BK = 128 / SZ;     // k values of a slice
  static constexpr int BYTES = R * 128;
  static constexpr int LOADS = R / 8 / NW;
  static constexpr int NC = R * SZ / 16;  // chunks of a k-outer row
  static constexpr int READS = KOUTER ? (SZ == 2 ? 2 : 4) : 1;  // a fragment
  static_assert(R % (8 * NW) == 0, "whole loads for every wave");

  const char* base;
  long ld_bytes;
  uint32_t off[LOADS];
  int extent;  // rows of the operand from this tile's first on
  int kend;
  const char* at;  // k-outer: where the next slice starts, and
  long left;       // the bytes from there on
  Rsrc rsrc;

  __device__ __forceinline__ void init(const T* p, long ld, int r0, int rows,
                                       int kend_, int wave, int lane) {
    ld_bytes = ld * SZ;
    extent = rows - r0;
    kend = kend_;
    if constexpr (KOUTER) {
      base = reinterpret_cast<const char*>(p) + (long)r0 * SZ;
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        const int at = (j * NW + wave) * 64 + lane;
        const int k = at / NC;
        const int c = (at % NC) ^ swizzle(k);
        off[j] = (uint32_t)(k * ld_bytes + c * 16);
      }
    } else {
      base = reinterpret_cast<const char*>(p) + (long)r0 * ld_bytes;
      const int c = (lane & 7) ^ (lane >> 3);
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        const int r = (j * NW + wave) * 8 + (lane >> 3);
        off[j] = (uint32_t)(r * ld_bytes + c * 16);
      }
    }
  }

  __device__ __forceinline__ static int swizzle(int k) {
    if constexpr (SZ == 2) {
      return (((k & 3) | (((k >> 3) & 3) << 2)) << 1) & (NC - 1);
    } else {
      return (((k >> 2) & 3) << 2) & (NC - 1);
    }
  }

  // Which buffer the next slice is loaded from: a k-outer operand's starts at
  // that slice's first row, so offsets within it stay small.
  __device__ __forceinline__ void start(int kbeg) {
    if constexpr (KOUTER) {
      at = base + (long)kbeg * ld_bytes;
      left = (long)(kend - kbeg - 1) * ld_bytes + (long)extent * SZ;
      rsrc = make_rsrc(at, left);
    } else {
      const int rows = extent < R ? extent : R;
      rsrc = make_rsrc(base, (long)(rows - 1) * ld_bytes + (long)kend * SZ);
    }
  }

  __device__ __forceinline__ void next() {
    if constexpr (KOUTER) {
      at += BK * ld_bytes;
      left -= BK * ld_bytes;
      rsrc = make_rsrc(at, left);
    }
  }

  // start load j of the slice at k0 into `lds`
  __device__ __forceinline__ void load(char* lds, int k0, int j, int wave,
                                       int lane) const {
    char* to = lds + (j * NW + wave) * 1024;
    if constexpr (KOUTER) {
      load_to_lds(rsrc, to, off[j], 0);
    } else {
      const int c = (lane & 7) ^ (lane >> 3);
      load_to_lds(rsrc, to, k0 + c * E >= kend ? OUT_OF_RANGE : off[j],
                  k0 * SZ);
    }
  }

  // the fragment of rows row0 .. row0+15, half `ks` of the slice
  __device__ __forceinline__ static Frag read(const char* lds, int row0,
                                              int ks, int lane) {
    Frag v;
    const int i = lane & 15, g = lane >> 4;
    if constexpr (!KOUTER) {
      const int c = (ks * 4 + g) ^ (i & 7);
      v.h = *reinterpret_cast<const s16x8*>(lds + (row0 + i) * 128 + c * 16);
    } else if constexpr (SZ == 2) {
      const int k = ks * 32 + g * 8 + (i >> 2);
      const int c = ((row0 >> 3) + ((i >> 1) & 1)) ^ swizzle(k);
      const char* p = lds + k * (R * 2) + c * 16 + (i & 1) * 8;
      v.q[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
      v.q[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_s16x4*)(p + 4 * (R * 2)));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = ks * 16 + g * 4 + j;
        const int c = ((row0 + i) >> 2) ^ swizzle(k);
        v.w[j] = *reinterpret_cast<const float*>(lds + k * (R * 4) + c * 16 +
                                                 (i & 3) * 4);
      }
    }
    return v;
  }
};

// acc (f32x4 [S::MI][S::NI]) += the product over k in [kbeg, kend); kbeg is a
// multiple of BK.  A k-inner operand needs whole chunks up to kend; rows of a
// k-outer one from `krows` on are taken for zeros.  `smem` is S::LDS bytes.
// begin() sets acc, while the first slices are on their way.  Every wave of the
// workgroup calls it with the same arguments; on return all of them are done
// with smem.
template <class T, bool KA, bool KB, class S, class Acc, class Begin>
__device__ __forceinline__ void product(const T* A, long lda, int m0, int M,
                                        const T* B, long ldb, int n0, int N,
                                        int kbeg, int kend, int krows,
                                        char* smem, Acc& acc, Begin begin) {
  using OA = Operand<T, KA, S::BM, S::NW>;
  using OB = Operand<T, KB, S::BN, S::NW>;
  constexpr int BK = OA::BK;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = (wave / S::WN) * (S::MI * 16);
  const int wn = (wave % S::WN) * (S::NI * 16);
  OA a;
  OB b;
  a.init(A, lda, m0, M, KA ? krows : kend, wave, lane);
  b.init(B, ldb, n0, N, KB ? krows : kend, wave, lane);

  // S::ST slices are in LDS or on their way there, and two halves of a slice
  // in registers: the matrix cores work on one half while the other is read.
  // Loads and reads past the last slice are harmless (zeros, unused), which
  // keeps the loop free of branches.
  Frag fa[2][S::MI], fb[2][S::NI];
  constexpr int FRAGS = S::MI + S::NI, LOADS = OA::LOADS + OB::LOADS;
  // one fragment of half ks; those of B first, the first products need them
  auto read = [&](const char* lds, int ks, int to, int i) {
    if (i < S::NI) {
      fb[to][i] = OB::read(lds + OA::BYTES, wn + i * 16, ks, lane);
    } else {
      fa[to][i - S::NI] = OA::read(lds, wm + (i - S::NI) * 16, ks, lane);
    }
  };
  auto multiply = [&](int from) {
#pragma unroll
    for (int mi = 0; mi < S::MI; ++mi) {
#pragma unroll
      for (int ni = 0; ni < S::NI; ++ni) {
        acc[mi][ni] = mma<T>(fa[from][mi], fb[from][ni], acc[mi][ni]);
      }
    }
  };
  auto load = [&](char* lds, int k0, int j) {
    if (j < OA::LOADS) {
      a.load(lds, k0, j, wave, lane);
    } else {
      b.load(lds + OA::BYTES, k0, j - OA::LOADS, wave, lane);
    }
  };
  a.start(kbeg);
  b.start(kbeg);
  int issued = kbeg;  // k of the next slice to be loaded
  auto load_slice = [&](char* lds) {
#pragma unroll
    for (int j = 0; j < LOADS; ++j) load(lds, issued, j);
    a.next();
    b.next();
    issued += BK;
  };
#pragma unroll
  for (int t = 0; t < S::ST; ++t) load_slice(smem + t * S::SLICE);
  begin();
  arrive<(S::ST - 1) * LOADS>();
  char* cur = smem;
#pragma unroll
  for (int i = 0; i < FRAGS; ++i) read(cur, 0, 0, i);
  for (int k0 = kbeg; k0 < kend; k0 += BK) {
    char* nxt = cur + S::SLICE;
    if (nxt == smem + S::LDS) nxt = smem;
#pragma unroll
    for (int i = 0; i < FRAGS; ++i) read(cur, 1, 1, i);
    multiply(0);
    spread<S::MI * S::NI * MMAS<T>, S::MI * OA::READS + S::NI * OB::READS>();
    // cur is in registers, nxt in LDS
    arrive<(S::ST - 2) * LOADS>();
    // the compiler keeps reads and loads, both of LDS, in this order
#pragma unroll
    for (int i = 0; i < (FRAGS > LOADS ? FRAGS : LOADS); ++i) {
      if (i < FRAGS) read(nxt, 0, 0, i);
      if (i < LOADS) load(cur, issued, i);
    }
    issued += BK;
    a.next();
    b.next();
    multiply(1);
    spread<S::MI * S::NI * MMAS<T>, S::MI * OA::READS + S::NI * OB::READS>();
    cur = nxt;
  }
  arrive<0>();
}

// Writes 16 columns of a wave's part of C, ROWS rows each, as rows of memory:
// out[j * ld + c] for column j and row c.  A lane holds 4 neighbouring rows of
// one column, v[ROWS / 16][4]; written from there, a store would be pieces of
// 32 bytes.  They go through LDS (`lds`, the wave's own, ROWS * 16 values) and
// leave as whole rows, one Unit a lane.  `cols` columns and `rows` rows exist
// (rows, out and ld in whole Units).
struct alignas(16) Chunk16 {
  int v[4];
};

template <class T, int ROWS, class Unit = Chunk16>
__device__ __forceinline__ void store_columns(const T (&v)[ROWS / 16][4],
                                              char* lds, T* out, long ld,
                                              int cols, int rows, int lane) {
  constexpr int E = 16 / sizeof(T), CH = ROWS / E, LINE = ROWS * sizeof(T);
  constexpr int UNITS = LINE / sizeof(Unit);       // of a column
  constexpr int SHARE = 16 / sizeof(Unit), EACH = sizeof(Unit) / sizeof(T);
  static_assert(16 * UNITS % 64 == 0, "whole stores");
  const int i = lane & 15, g = lane >> 4;
#pragma unroll
  for (int m = 0; m < ROWS / 16; ++m) {
    const int at = m * 16 + g * 4;
    __builtin_memcpy(lds + i * LINE + (((at / E) ^ (i & (CH - 1))) * 16) +
                         (at % E) * sizeof(T),
                     v[m], 4 * sizeof(T));
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int q = 0; q < 16 * UNITS / 64; ++q) {
    const int j = (q * 64 + lane) / UNITS, c = (q * 64 + lane) % UNITS;
    const Unit t = *reinterpret_cast<const Unit*>(
        lds + j * LINE + (((c / SHARE) ^ (j & (CH - 1))) * 16) +
        (c % SHARE) * sizeof(Unit));
    if (j < cols && c * EACH < rows) {
      *reinterpret_cast<Unit*>(out + (long)j * ld + c * EACH) = t;
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Which tile of mt x nt workgroup `id` takes; false: none.  Workgroups go to
// the 8 XCDs in turn; each XCD has an L2 of its own, so each gets one run of
// neighbouring tiles, and a run walks 8 tiles of m for each tile of n before
// the next n.  nt is of the rows that are there (a count on the device): were
// it of the rows that there may be, some XCDs would get most of the work.
__device__ __forceinline__ bool pick(int id, int mt, int nt, int* m, int* n) {
  const int total = mt * nt;
  if (id >= total) return false;
  const int q = total >> 3, r = total & 7;
  const int x = id & 7, y = id >> 3;
  const int p = x * q + (x < r ? x : r) + y;
  const int group = p / (8 * nt);
  const int first = group * 8;
  const int wide = mt - first < 8 ? mt - first : 8;
  const int in = p - first * nt;
  *m = first + in % wide;
  *n = in / wide;
  return true;
}

}  // namespace tile
