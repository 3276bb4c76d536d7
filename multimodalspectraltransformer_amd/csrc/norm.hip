// Dropout from a counter-based generator and layer norm of any width (forward, backward, optional residual and dropout in
// front of it): the row operators of a post-norm or pre-norm block outside the width-128 fused launches.
//
//   dropout     y = keep(seed, offset, i) ? x * 65536 / (65536 - thr) : 0            (philox.h; its backward is itself)
//   layer norm  z = residual + dropout(x),  y = (z - mean) rstd gamma + beta
//               q = dy gamma,  xh = (z - mean) rstd,  dz = rstd (q - mean(q) - xh mean(q xh)) + dz_in,  dx = dropout(dz)
//               dgamma = sum over rows of dy xh,  dbeta = sum over rows of dy
//
// All of it is bound by HBM: every tensor is read or written once and a row stays in registers between the statistics and
// the output.  TPR lanes own a row (4 lanes for 32 columns up to a workgroup of 1024 for 16384), NV groups of eight
// columns each, so that a lane's accesses are 16 bytes wide, whatever their alignment; the last group of a row whose width
// is no multiple of eight is read as the last eight columns and moved.
#include "../../include/mmst.h"
#include "philox.h"

namespace {

typedef _Float16 f16;
template <typename T> struct Vec8 { T v[8]; } __attribute__((aligned(16)));

// Eight elements as 16-byte accesses at any alignment of an element: the hardware takes them (a wave's 1 KiB touches one
// more cache line then), so rows of odd widths and strides need no form of their own.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <int A> struct __attribute__((packed, aligned(A))) Packed16 { u32x4 v; };
template <typename T> __device__ __forceinline__ void load_vec(Vec8<T>& d, const T* p) {
  constexpr int N = sizeof(Vec8<T>) / 16;
  u32x4 u[N];
#pragma unroll
  for (int i = 0; i < N; ++i) u[i] = reinterpret_cast<const Packed16<sizeof(T)>*>(p)[i].v;
  __builtin_memcpy(&d, u, sizeof d);
}
template <typename T> __device__ __forceinline__ void store_vec(T* p, const float (&v)[8]) {
  Vec8<T> d;
#pragma unroll
  for (int e = 0; e < 8; ++e) d.v[e] = (T)v[e];
  constexpr int N = sizeof(Vec8<T>) / 16;
  u32x4 u[N];
  __builtin_memcpy(u, &d, sizeof d);
#pragma unroll
  for (int i = 0; i < N; ++i) reinterpret_cast<Packed16<sizeof(T)>*>(p)[i].v = u[i];
}

// ---------------------------------------------------------------------------------------------------- dropout
struct DropArgs {
  const void* x; void* y;
  uint64_t n, cols, ldx, ldy;   // n = rows * cols
  uint64_t wg0;                 // workgroups of the launches before this one
  DropKey key;
};

// A lane owns blocks of eight elements.  FLAT: rows follow one another, and the tensor is one row.  ROWS: rows of a multiple of
// eight elements, a block lies inside one.  ANY: of eight elements or more; a block may begin in one row and end in the next,
// and goes by elements then.  37248 x 2048 in bf16 (FLAT): 56 us, 5.4 TB/s, as fast as a copy; two blocks per lane of a 16-bit
// type keep 32 bytes per lane in flight as one does of fp32.
enum { FLAT = 0, ROWS = 1, ANY = 2 };
template <typename T, int MODE, int U>
__global__ __launch_bounds__(256) void dropout_vec_kernel(const DropArgs a) {
  const uint64_t nb = MODE == ANY ? (a.n + 7) >> 3 : a.n >> 3;
  const uint64_t b0 = (a.wg0 + blockIdx.x) * (256 * U) + threadIdx.x;
  Vec8<T> in[U];
  uint64_t ox[U], oy[U];
  int left[U];   // elements before the end of the row (ANY)
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint64_t b = b0 + 256 * u;
    if (b >= nb) continue;
    ox[u] = oy[u] = b << 3;
    left[u] = 8;
    if constexpr (MODE != FLAT) {
      const uint64_t i = b << 3, r = (a.n >> 32) ? i / a.cols : (uint64_t)((uint32_t)i / (uint32_t)a.cols), c = i - r * a.cols;
      ox[u] = r * a.ldx + c;
      oy[u] = r * a.ldy + c;
      if constexpr (MODE == ANY) left[u] = a.cols - c < 8 ? (int)(a.cols - c) : 8;
    }
    if (MODE != ANY || left[u] == 8) {
      load_vec(in[u], (const T*)a.x + ox[u]);
    } else {
      const T* p = (const T*)a.x + ox[u];
#pragma unroll
      for (int e = 0; e < 8; ++e) in[u].v[e] = (b << 3) + e < a.n ? p[e < left[u] ? (uint64_t)e : e + a.ldx - a.cols] : (T)0.f;
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint64_t b = b0 + 256 * u;
    if (b >= nb) continue;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)in[u].v[e];
    if (a.key.thr) drop_block(v, philox_block(b, a.key), a.key);
    if (MODE != ANY || left[u] == 8) {
      store_vec((T*)a.y + oy[u], v);
    } else {
      T* p = (T*)a.y + oy[u];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if ((b << 3) + e < a.n) p[e < left[u] ? (uint64_t)e : e + a.ldy - a.cols] = (T)v[e];
    }
  }
  if constexpr (MODE == FLAT) {   // the last n % 8 elements
    const uint64_t i = (nb << 3) + threadIdx.x;
    if (blockIdx.x == 0 && a.wg0 == 0 && i < a.n) {
      const uint4 w = philox_block(nb, a.key);
      const uint32_t word = threadIdx.x < 2 ? w.x : threadIdx.x < 4 ? w.y : threadIdx.x < 6 ? w.z : w.w;
      const uint32_t bits = threadIdx.x & 1 ? word >> 16 : word & 0xFFFFu;
      const float v = (float)((const T*)a.x)[i];
      ((T*)a.y)[i] = (T)(bits >= a.key.thr ? v * a.key.scale : 0.f);
    }
  }
}

// short rows of an odd width that do not follow one another, so that a block may lie in two or more: a wave owns 512
// consecutive elements, a lane one element per access
template <typename T>
__global__ __launch_bounds__(256) void dropout_elem_kernel(const DropArgs a) {
  __shared__ uint4 slots[4][65];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t first = ((a.wg0 + blockIdx.x) * 4 + wave) * 512;
  float v[8];
  uint64_t oy[8];
  uint64_t i = first + lane;
  uint64_t r = (a.n >> 32) ? i / a.cols : (uint64_t)((uint32_t)i / (uint32_t)a.cols);   // cols <= n
  uint64_t c = i - r * a.cols;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const bool ok = i < a.n;
    v[j] = ok ? (float)((const T*)a.x)[r * a.ldx + c] : 0.f;
    oy[j] = r * a.ldy + c;
    i += 64;
    c += 64;
    if (a.cols >= 64) {
      if (c >= a.cols) { c -= a.cols; ++r; }
    } else {
      r += (uint32_t)c / (uint32_t)a.cols;
      c = (uint32_t)c % (uint32_t)a.cols;
    }
  }
  if (a.key.thr) drop_elements<64>(v, first, a.key, slots[wave], lane);
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (first + j * 64 + lane < a.n) ((T*)a.y)[oy[j]] = (T)v[j];
}

// Rows of an odd width and a stride of their own: blocks from 32 columns of a 16-bit type and 128 of fp32 on, where few enough of
// them lie in two rows, single elements below.  Blocks / elements: bf16 17 columns 52 / 48 us, 41 39 / 46, 4099 25 / 46 (of 33 to
// 36 M elements), fp32 65 columns 55 / 43, 101 39.5 / 38, 501 39 / 43, 4099 41 / 44.
template <typename T> constexpr uint64_t any_cols() { return sizeof(T) == 2 ? 32 : 128; }

template <typename T> int launch_dropout(DropArgs& a, hipStream_t st) {
  const bool flat = a.ldx == a.cols && a.ldy == a.cols, rows = a.cols % 8 == 0, any = a.cols >= any_cols<T>();
  constexpr int U = sizeof(T) == 4 ? 1 : 2;
  const uint64_t all = flat || rows || any ? (a.n / 8 + 256 * U) / (256 * U) : (a.n + 2047) / 2048, most = 1u << 20;
  do {   // (a launch has less than 2^32 threads)
    const uint64_t left = all - a.wg0;
    const dim3 grid(left > most ? (unsigned)most : (unsigned)left);
    if (flat) hipLaunchKernelGGL((dropout_vec_kernel<T, FLAT, U>), grid, dim3(256), 0, st, a);
    else if (rows) hipLaunchKernelGGL((dropout_vec_kernel<T, ROWS, U>), grid, dim3(256), 0, st, a);
    else if (any) hipLaunchKernelGGL((dropout_vec_kernel<T, ANY, U>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((dropout_elem_kernel<T>), grid, dim3(256), 0, st, a);
    MMST_CHECK_LAUNCH();
    a.wg0 += most;
  } while (a.wg0 < all);
  return MMST_OK;
}

// ---------------------------------------------------------------------------------------------------- layer norm
struct LnArgs {
  const void* x; const void* res;           // forward: input, residual; backward: dy, dz_in
  const void* zin;                          // backward: z
  const float* gamma; const float* beta;
  void* y; void* z; float* stats;           // forward: y, z, statistics out; backward: dz, dx, statistics in
  float* part;                              // backward: [gridDim.x][2][cols] column sums of each workgroup
  long rows; int cols;
  long ldx, ldr, ldzin, ldy, ldz;
  float eps, inv_cols;
  DropKey key;
};

// sum over the TPR lanes that own a row, on all of them; wider than a wave: through LDS, two buffers in turn, so that one
// barrier per sum is enough (a buffer is written again only behind the next sum's barrier)
template <int TPR, int BLK> __device__ __forceinline__ float row_sum(float v, float (*red)[BLK / 64], int& turn) {
  if constexpr (TPR == 4) {
    v += dpp_f32<0xB1>(v);
    return v + dpp_f32<0x4E>(v);
  } else if constexpr (TPR == 8) return row8_sum(v);
  else if constexpr (TPR == 16) return row16_sum(v);
  else if constexpr (TPR == 32) return xor16_sum(row16_sum(v));
  else {
    v = wave_sum(v);
    if constexpr (TPR > 64) {
      float* r = red[turn];
      turn ^= 1;
      if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = v;
      __syncthreads();
      v = 0.f;
#pragma unroll
      for (int i = 0; i < TPR / 64; ++i) v += r[(threadIdx.x / TPR) * (TPR / 64) + i];
    }
    return v;
  }
}

// Group q of lane t of a row: columns (q * TPR + t) * 8 .. + 7.  ODD: cols is no multiple of eight, so one lane's last group is
// cut off.  It is loaded as the row's last eight columns, so that nothing behind the row is read, and moved down by the columns
// that belong to the lane before (ln_fix, when the loads of all tensors are under way: moving needs them).  Column by column:
// 153 us instead of 52 for the backward pass of 262000 x 127 in bf16.
template <int N> __device__ __forceinline__ void words_down(uint32_t (&w)[N], int by, bool go) {
#pragma unroll
  for (int i = 0; i < N; ++i) w[i] = go ? (i + by < N ? w[i + by] : 0u) : w[i];
}
template <typename T> __device__ __forceinline__ void move_down(Vec8<T>& d, int n) {   // n: 1..7 elements, the same in every lane
  constexpr int N = sizeof(Vec8<T>) / 4;
  uint32_t w[N];
  __builtin_memcpy(w, &d, sizeof d);
  words_down(w, N / 2, n & 4);
  words_down(w, N / 4, n & 2);
  if constexpr (N == 8) {
    words_down(w, 1, n & 1);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = n & 1 ? __builtin_amdgcn_alignbit(i + 1 < N ? w[i + 1] : 0u, w[i], 16) : w[i];
  }
  __builtin_memcpy(&d, w, sizeof d);
}
template <bool ODD> __device__ __forceinline__ int cut_off(int c, int cols) {   // columns that the group at c lacks
  return ODD && c + 8 > cols && cols >= 8 ? c + 8 - cols : 0;
}
template <typename T, bool ODD> __device__ __forceinline__ void load_group(Vec8<T>& d, const T* row, int c, int cols) {
  if (!ODD || cols >= 8) {
    load_vec(d, row + c - cut_off<ODD>(c, cols));
  } else {   // a row of less than eight columns
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < cols) d.v[e] = row[e];
  }
}
template <typename T, bool ODD, int TPR, int NV>
__device__ __forceinline__ void ln_load(Vec8<T> (&d)[NV], const T* row, int cols, int t, bool ok) {
#pragma unroll
  for (int q = 0; q < NV; ++q) {
    const int c = (q * TPR + t) * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) d[q].v[e] = (T)0.f;
    if (ok && c < cols) load_group<T, ODD>(d[q], row, c, cols);
  }
}
template <typename T, bool ODD, int TPR, int NV> __device__ __forceinline__ void ln_fix(Vec8<T> (&d)[NV], int cols, int t) {
  if constexpr (ODD)
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      const int c = (q * TPR + t) * 8;
      if (c < cols && cut_off<ODD>(c, cols)) move_down(d[q], 8 - (cols & 7));
    }
}
template <typename T, bool ODD, int TPR>
__device__ __forceinline__ void ln_store(T* row, const float (&v)[8], int cols, int q, int t) {
  const int c = (q * TPR + t) * 8;
  if (c + (ODD ? 7 : 0) < cols) {
    store_vec(row + c, v);
  } else if (ODD && c < cols) {   // four, two and one columns
    const int n = cols & 7;
    T* p = row + c;
    float w[4] = {v[0], v[1], v[2], v[3]};
    if (n & 4) {
#pragma unroll
      for (int e = 0; e < 4; ++e) { p[e] = (T)w[e]; w[e] = v[4 + e]; }
      p += 4;
    }
    if (n & 2) {
      p[0] = (T)w[0];
      p[1] = (T)w[1];
      w[0] = w[2];
      p += 2;
    }
    if (n & 1) p[0] = (T)w[0];
  }
}
template <bool ODD, int TPR>
__device__ __forceinline__ void ln_vec_f32(float (&v)[8], const float* p, float none, int cols, int q, int t) {
  const int c = (q * TPR + t) * 8;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = none;
  if (p && c < cols) {
    Vec8<float> d = {};
    load_group<float, ODD>(d, p, c, cols);
    if (cut_off<ODD>(c, cols)) move_down(d, 8 - (cols & 7));
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = d.v[e];
  }
}
// dropout of group q of row r, whose elements are r * cols + column of the tensor read row by row
template <bool ODD, int TPR>
__device__ __forceinline__ void ln_drop(float (&v)[8], const DropKey& k, long r, int cols, int q, int t, uint4* slots) {
  if constexpr (!ODD) {
    drop_block(v, philox_block((uint64_t)r * (uint64_t)(cols >> 3) + (uint64_t)(q * TPR + t), k), k);
  } else {
    constexpr int G = TPR < 64 ? TPR : 64;
    drop_straddling<G>(v, (uint64_t)r * cols + (uint64_t)((q * TPR + (t / G) * G) * 8), k,
                       slots + (threadIdx.x / G) * (G + 1), t % G);
  }
}

template <typename T, bool ODD, int TPR, int NV, int BLK>
__global__ __launch_bounds__(BLK) void ln_fwd_kernel(const LnArgs a) {
  constexpr int RPB = BLK / TPR, G = TPR < 64 ? TPR : 64;
  __shared__ float red[2][BLK / 64];
  __shared__ uint4 slots[!ODD ? 1 : (BLK / G) * (G + 1)];
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR, cols = a.cols;
  int turn = 0;
  for (long base = (long)blockIdx.x * RPB; base < a.rows; base += (long)gridDim.x * RPB) {
    const long r = base + sub;
    const bool ok = r < a.rows;
    Vec8<T> x[NV], rs[NV];
    ln_load<T, ODD, TPR, NV>(x, (const T*)a.x + r * a.ldx, cols, t, ok);
    if (a.res) ln_load<T, ODD, TPR, NV>(rs, (const T*)a.res + r * a.ldr, cols, t, ok);
    ln_fix<T, ODD, TPR, NV>(x, cols, t);
    if (a.res) ln_fix<T, ODD, TPR, NV>(rs, cols, t);
    float z[NV][8];
    float s = 0.f;
#pragma unroll
    for (int q = 0; q < NV; ++q) {
#pragma unroll
      for (int e = 0; e < 8; ++e) z[q][e] = (float)x[q].v[e];
      if (a.key.thr) ln_drop<ODD, TPR>(z[q], a.key, r, cols, q, t, slots);
      if (a.res)
#pragma unroll
        for (int e = 0; e < 8; ++e) z[q][e] += (float)rs[q].v[e];
#pragma unroll
      for (int e = 0; e < 8; ++e) s += z[q][e];   // columns past the end are zero
    }
    // (a product with 1 / cols would not leave a constant row at 0)
    const float mean = row_sum<TPR, BLK>(s, red, turn) / (float)cols;
    float vs = 0.f;   // the variance from the centred row: a large mean costs no digits
#pragma unroll
    for (int q = 0; q < NV; ++q)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = (q * TPR + t) * 8 + (ODD ? e : 0) < cols ? z[q][e] - mean : 0.f;
        vs += d * d;
      }
    const float rstd = 1.0f / sqrtf(row_sum<TPR, BLK>(vs, red, turn) / (float)cols + a.eps);
    if (ok) {
#pragma unroll
      for (int q = 0; q < NV; ++q) {
        if (a.z) ln_store<T, ODD, TPR>((T*)a.z + r * a.ldz, z[q], cols, q, t);
        float g[8], b[8], y[8];
        ln_vec_f32<ODD, TPR>(g, a.gamma, 1.f, cols, q, t);
        ln_vec_f32<ODD, TPR>(b, a.beta, 0.f, cols, q, t);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = (z[q][e] - mean) * rstd * g[e] + b[e];
        ln_store<T, ODD, TPR>((T*)a.y + r * a.ldy, y, cols, q, t);
      }
      if (t == 0 && a.stats) { a.stats[2 * r] = mean; a.stats[2 * r + 1] = rstd; }
    }
  }
}

template <typename T, bool ODD, int TPR, int NV, int BLK>
__global__ __launch_bounds__(BLK) void ln_bwd_kernel(const LnArgs a) {
  constexpr int RPB = BLK / TPR, G = TPR < 64 ? TPR : 64, CAP = TPR * NV * 8;
  __shared__ float red[2][BLK / 64];
  __shared__ uint4 slots[!ODD ? 1 : (BLK / G) * (G + 1)];
  __shared__ float sums[RPB > 1 ? RPB * CAP : 1];
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR, cols = a.cols;
  int turn = 0;
  float pg[NV][8], pb[NV][8];
#pragma unroll
  for (int q = 0; q < NV; ++q)
#pragma unroll
    for (int e = 0; e < 8; ++e) pg[q][e] = pb[q][e] = 0.f;
  for (long base = (long)blockIdx.x * RPB; base < a.rows; base += (long)gridDim.x * RPB) {
    const long r = base + sub;
    const bool ok = r < a.rows;
    Vec8<T> dy[NV], zv[NV], add[NV];
    ln_load<T, ODD, TPR, NV>(dy, (const T*)a.x + r * a.ldx, cols, t, ok);
    ln_load<T, ODD, TPR, NV>(zv, (const T*)a.zin + r * a.ldzin, cols, t, ok);
    if (a.res) ln_load<T, ODD, TPR, NV>(add, (const T*)a.res + r * a.ldr, cols, t, ok);
    const float mean = ok ? a.stats[2 * r] : 0.f, rstd = ok ? a.stats[2 * r + 1] : 0.f;
    ln_fix<T, ODD, TPR, NV>(dy, cols, t);
    ln_fix<T, ODD, TPR, NV>(zv, cols, t);
    if (a.res) ln_fix<T, ODD, TPR, NV>(add, cols, t);
    float xh[NV][8], qv[NV][8];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      float g[8];
      ln_vec_f32<ODD, TPR>(g, a.gamma, 1.f, cols, q, t);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = (float)dy[q].v[e];   // zero past the last column and row, so every sum is
        xh[q][e] = ((float)zv[q].v[e] - mean) * rstd;
        qv[q][e] = d * g[e];
        s1 += qv[q][e];
        s2 += qv[q][e] * xh[q][e];
        pg[q][e] += d * xh[q][e];
        pb[q][e] += d;
      }
    }
    s1 = row_sum<TPR, BLK>(s1, red, turn) * a.inv_cols;
    s2 = row_sum<TPR, BLK>(s2, red, turn) * a.inv_cols;
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      float dz[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) dz[e] = rstd * (qv[q][e] - s1 - xh[q][e] * s2);
      if (a.res)
#pragma unroll
        for (int e = 0; e < 8; ++e) dz[e] += (float)add[q].v[e];
      if (ok) ln_store<T, ODD, TPR>((T*)a.y + r * a.ldy, dz, cols, q, t);
      if (a.key.thr) {   // (every lane: the lanes of a row share the generator's words)
        ln_drop<ODD, TPR>(dz, a.key, r, cols, q, t, slots);
        if (ok) ln_store<T, ODD, TPR>((T*)a.z + r * a.ldz, dz, cols, q, t);
      }
    }
  }
  if (!a.part) return;
  // column sums of the workgroup's rows: its row groups one after another, in a fixed order
  float* part = a.part + (size_t)blockIdx.x * 2 * cols;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    if constexpr (RPB == 1) {
#pragma unroll
      for (int q = 0; q < NV; ++q)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int c = (q * TPR + t) * 8 + e;
          if (c < cols) part[w * cols + c] = w ? pb[q][e] : pg[q][e];
        }
    } else {
      __syncthreads();
#pragma unroll
      for (int q = 0; q < NV; ++q)
#pragma unroll
        for (int e = 0; e < 8; ++e) sums[sub * CAP + (q * TPR + t) * 8 + e] = w ? pb[q][e] : pg[q][e];
      __syncthreads();
      for (int c = threadIdx.x; c < cols; c += BLK) {
        float s = 0.f;
#pragma unroll 4
        for (int i = 0; i < RPB; ++i) s += sums[i * CAP + c];
        part[w * cols + c] = s;
      }
    }
  }
}

// dgamma / dbeta = sum over the n workgroups' column sums, in order: 16 columns per workgroup, 64 slices of the rows, so
// that the up to 512 rows of a narrow layer norm are 8 loads deep (4.3 us; with 64 columns and 16 slices 6.0 us)
__global__ __launch_bounds__(1024) void ln_cols_kernel(const float* part, int n, int cols, float* dgamma, float* dbeta,
                                                       int accumulate) {
  __shared__ float red[64][17];
  const int lane = threadIdx.x & 15, w = threadIdx.x >> 4;
  const long c = (long)blockIdx.x * 16 + lane;
  float s = 0.f;
  if (c < 2L * cols) {
#pragma unroll 4
    for (int i = w; i < n; i += 64) s += part[(size_t)i * 2 * cols + c];
  }
  red[w][lane] = s;
  __syncthreads();
  if (w < 16) {   // transposed: 16 lanes per column, four slices each
    s = red[4 * lane][w] + red[4 * lane + 1][w] + red[4 * lane + 2][w] + red[4 * lane + 3][w];
    s = row16_sum(s);
    const long k = (long)blockIdx.x * 16 + w;
    if (lane == 0 && k < 2L * cols) {
      float* out = k < cols ? (dgamma ? dgamma + k : nullptr) : (dbeta ? dbeta + (k - cols) : nullptr);
      if (out) *out = accumulate ? *out + s : s;
    }
  }
}

struct LnShape { int tpr, nv, blk, grid; };

// Lanes per row: as few as hold it with a few accesses each, so that a wave has several rows' loads in flight and few idle
// lanes.  Forward with a residual, bf16, one shape / the next: 1000000 x 24 4 lanes 32 us, 16 90; 524288 x 64 8 lanes 45, 16 59;
// 262144 x 128 16 lanes 45, 32 58; 60000 x 520 32 lanes with three accesses 43, 64 with two 50; 25000 x 1200 64 lanes with three
// 39, 256 with one 47; 16000 x 2048 256 with one 41, 64 with four 42; 8000 x 4099 256 with three 67, with four 92; 4096 x 8192
// 256 with four 44, 1024 with two 57.  6 TB/s of bf16 and 5 of fp32 at even widths that fill their lanes.  Workgroups take rows
// in turn beyond 4096 (2048: up to 10 % slower for odd widths, which wait longer per row).
LnShape ln_fwd_shape(long rows, int cols) {
  LnShape s;
  s.blk = cols <= 8192 ? 256 : 1024;
  s.tpr = cols <= 32 ? 4 : cols <= 64 ? 8 : cols <= 128 ? 16 : cols <= 768 ? 32 : cols <= 1536 ? 64 : cols <= 8192 ? 256 : 1024;
  s.nv = (cols + s.tpr * 8 - 1) / (s.tpr * 8);
  if (s.tpr == 1024) s.nv = 2;
  const long need = (rows + s.blk / s.tpr - 1) / (s.blk / s.tpr);
  s.grid = (int)(need < 4096 ? need : 4096);
  return s;
}
// The backward pass keeps two sums per column besides the row, and each workgroup leaves them for ln_cols_kernel: two
// workgroups of 256 per CU, or one of 1024 (four and two: 5 % faster to 7 % slower, and 15 to 45 % slower from 4096 columns
// on, where the sums themselves are most of what is written).  Up to 1536 columns lanes as above, in a wave (60000 x 520
// bf16: 32 lanes with three accesses 38 us, 64 with two 43; 25000 x 1200: 64 with three 35, 256 of a larger workgroup 42).
// Beyond, two accesses per lane only where the 128 registers of a 1024-lane workgroup hold that (16-bit types, even widths:
// 8192 x 4096 39 us, 42 with one; 4096 x 8192 43 and 53; two accesses in workgroups of 256 at 8000 x 4099 88, one in a
// workgroup of 1024 79), or where there is no wider workgroup.
LnShape ln_bwd_shape(long rows, int cols, int dtype) {
  LnShape s;
  const bool one = cols % 8 || dtype == MMST_F32;
  s.blk = cols <= 1536 ? 256 : 1024;
  s.tpr = cols <= 32 ? 4 : cols <= 64 ? 8 : cols <= 128 ? 16 : cols <= 768 ? 32 : cols <= 1536 ? 64 : cols <= 2048 ? 256
        : cols <= 4096 ? (one ? 512 : 256) : cols <= 8192 ? (one ? 1024 : 512) : 1024;
  s.nv = (cols + s.tpr * 8 - 1) / (s.tpr * 8);
  const long need = (rows + s.blk / s.tpr - 1) / (s.blk / s.tpr), most = s.blk == 256 ? 512 : 256;
  s.grid = (int)(need < most ? need : most);
  return s;
}

#define LN_CASE(K, TPR, NV, BLK)                                                                     \
  if (s.tpr == TPR && s.nv == NV && s.blk == BLK) {                                                 \
    if (a.cols % 8) hipLaunchKernelGGL((K<T, true, TPR, NV, BLK>), dim3(s.grid), dim3(BLK), 0, st, a); \
    else hipLaunchKernelGGL((K<T, false, TPR, NV, BLK>), dim3(s.grid), dim3(BLK), 0, st, a);        \
    return true;                                                                                    \
  }
#define LN_WIDE(TPR)                                                                                 \
  if (s.tpr == TPR && s.nv == 2) {                                                                  \
    hipLaunchKernelGGL((ln_bwd_kernel<T, false, TPR, 2, 1024>), dim3(s.grid), dim3(1024), 0, st, a); \
    return true;                                                                                    \
  }
// (false: a shape without a kernel)
template <typename T> bool launch_ln_fwd(const LnArgs& a, const LnShape& s, hipStream_t st) {
  LN_CASE(ln_fwd_kernel, 4, 1, 256)
  LN_CASE(ln_fwd_kernel, 8, 1, 256)
  LN_CASE(ln_fwd_kernel, 16, 1, 256)
  LN_CASE(ln_fwd_kernel, 32, 1, 256)
  LN_CASE(ln_fwd_kernel, 32, 2, 256)
  LN_CASE(ln_fwd_kernel, 32, 3, 256)
  LN_CASE(ln_fwd_kernel, 64, 2, 256)
  LN_CASE(ln_fwd_kernel, 64, 3, 256)
  LN_CASE(ln_fwd_kernel, 256, 1, 256)
  LN_CASE(ln_fwd_kernel, 256, 2, 256)
  LN_CASE(ln_fwd_kernel, 256, 3, 256)
  LN_CASE(ln_fwd_kernel, 256, 4, 256)
  LN_CASE(ln_fwd_kernel, 1024, 2, 1024)
  return false;
}
template <typename T> bool launch_ln_bwd(const LnArgs& a, const LnShape& s, hipStream_t st) {
  LN_CASE(ln_bwd_kernel, 4, 1, 256)
  LN_CASE(ln_bwd_kernel, 8, 1, 256)
  LN_CASE(ln_bwd_kernel, 16, 1, 256)
  LN_CASE(ln_bwd_kernel, 32, 1, 256)
  LN_CASE(ln_bwd_kernel, 32, 2, 256)
  LN_CASE(ln_bwd_kernel, 32, 3, 256)
  LN_CASE(ln_bwd_kernel, 64, 2, 256)
  LN_CASE(ln_bwd_kernel, 64, 3, 256)
  LN_CASE(ln_bwd_kernel, 256, 1, 1024)
  LN_CASE(ln_bwd_kernel, 1024, 2, 1024)
  if constexpr (sizeof(T) == 2)
    if (a.cols % 8 == 0) {
      LN_WIDE(256)
      LN_WIDE(512)
    }
  LN_CASE(ln_bwd_kernel, 512, 1, 1024)
  LN_CASE(ln_bwd_kernel, 1024, 1, 1024)
  return false;
}
#undef LN_CASE
#undef LN_WIDE

bool drop_ok(double p) { return p >= 0.0 && p <= 1.0; }   // (false for NaN)
bool type_ok(int dtype) { return dtype == MMST_F32 || dtype == MMST_BF16 || dtype == MMST_F16; }
bool ld_ok(const void* p, long ld, long cols, long rows) { return !p || rows <= 1 || ld >= cols; }

}  // namespace

extern "C" {

int mmst_dropout(const void* x, long ldx, void* y, long ldy, int dtype, long rows, long cols, double p, uint64_t seed,
                 uint64_t offset, void* stream) {
  if (!type_ok(dtype) || rows < 0 || cols < 0 || !drop_ok(p)) return MMST_ERR_ARG;
  if (rows == 0 || cols == 0) return MMST_OK;
  if (!x || !y || !ld_ok(x, ldx, cols, rows) || !ld_ok(y, ldy, cols, rows)) return MMST_ERR_ARG;
  if (rows > (long)(0x7FFFFFFFFFFFL / cols)) return MMST_ERR_ARG;
  if (rows == 1) ldx = ldy = cols;
  DropArgs a{x, y, (uint64_t)rows * (uint64_t)cols, (uint64_t)cols, (uint64_t)ldx, (uint64_t)ldy, 0, drop_key(p, seed, offset)};
  if (dtype == MMST_F32) return launch_dropout<float>(a, (hipStream_t)stream);
  if (dtype == MMST_BF16) return launch_dropout<bf16>(a, (hipStream_t)stream);
  return launch_dropout<f16>(a, (hipStream_t)stream);
}

int mmst_layer_norm(const void* x, long ldx, const void* residual, long ldr, const float* gamma, const float* beta, void* y,
                    long ldy, void* z, long ldz, float* stats, int dtype, long rows, int cols, float eps, double p,
                    uint64_t seed, uint64_t offset, void* stream) {
  if (!type_ok(dtype) || rows < 0 || cols < 1 || cols > MMST_LN_MAX_COLS || !drop_ok(p) || !(eps >= 0.f)) return MMST_ERR_ARG;
  if (rows == 0) return MMST_OK;
  if (!x || !y || !ld_ok(x, ldx, cols, rows) || !ld_ok(residual, ldr, cols, rows) || !ld_ok(y, ldy, cols, rows) ||
      !ld_ok(z, ldz, cols, rows) || rows > 0x7FFFFFFFFFFFL / cols || y == z)
    return MMST_ERR_ARG;
  LnArgs a{x, residual, nullptr, gamma, beta, y, z, stats, nullptr, rows, cols, ldx, ldr, 0, ldy, ldz,
           eps, 1.0f / (float)cols, drop_key(p, seed, offset)};
  const LnShape s = ln_fwd_shape(rows, cols);
  const hipStream_t st = (hipStream_t)stream;
  if (!(dtype == MMST_F32 ? launch_ln_fwd<float>(a, s, st) : dtype == MMST_BF16 ? launch_ln_fwd<bf16>(a, s, st)
                                                                                 : launch_ln_fwd<f16>(a, s, st)))
    return MMST_ERR_LAUNCH;
  MMST_CHECK_LAUNCH();
  return MMST_OK;
}

int mmst_layer_norm_bwd_ws(int dtype, long rows, int cols, size_t* bytes) {
  if (!bytes || !type_ok(dtype) || rows < 0 || cols < 1 || cols > MMST_LN_MAX_COLS) return MMST_ERR_ARG;
  *bytes = (size_t)ln_bwd_shape(rows, cols, dtype).grid * 2 * cols * sizeof(float);
  return MMST_OK;
}

int mmst_layer_norm_bwd(const void* dy, long lddy, const void* z, long ldz, const float* stats, const float* gamma,
                        const void* dz_in, long lddz_in, void* dz, long lddz, void* dx, long lddx, float* dgamma,
                        float* dbeta, int accumulate, int dtype, long rows, int cols, double p, uint64_t seed,
                        uint64_t offset, void* ws, size_t ws_bytes, void* stream) {
  if (!type_ok(dtype) || rows < 0 || cols < 1 || cols > MMST_LN_MAX_COLS || !drop_ok(p)) return MMST_ERR_ARG;
  const LnShape s = ln_bwd_shape(rows, cols, dtype);
  const bool sums = dgamma || dbeta;
  if (sums && ws_bytes < (size_t)s.grid * 2 * cols * sizeof(float)) return MMST_ERR_ARG;
  if (dgamma && dbeta && dgamma < dbeta + cols && dbeta < dgamma + cols) return MMST_ERR_ARG;
  if (rows > 0) {
    const DropKey key = drop_key(p, seed, offset);
    if (!dy || !z || !stats || !dz || (key.thr && !dx) || (sums && (!ws || (uintptr_t)ws % 4)) || !ld_ok(dy, lddy, cols, rows) ||
        !ld_ok(z, ldz, cols, rows) || !ld_ok(dz_in, lddz_in, cols, rows) || !ld_ok(dz, lddz, cols, rows) ||
        !ld_ok(key.thr ? dx : nullptr, lddx, cols, rows) || (key.thr && dx == dz) || rows > 0x7FFFFFFFFFFFL / cols)
      return MMST_ERR_ARG;
    LnArgs a{dy, dz_in, z, gamma, nullptr, dz, dx, const_cast<float*>(stats), sums ? (float*)ws : nullptr, rows, cols,
             lddy, lddz_in, ldz, lddz, lddx, 0.f, 1.0f / (float)cols, key};
    const hipStream_t st = (hipStream_t)stream;
    if (!(dtype == MMST_F32 ? launch_ln_bwd<float>(a, s, st) : dtype == MMST_BF16 ? launch_ln_bwd<bf16>(a, s, st)
                                                                                   : launch_ln_bwd<f16>(a, s, st)))
      return MMST_ERR_LAUNCH;
    MMST_CHECK_LAUNCH();
  }
  if (sums) {
    hipLaunchKernelGGL(ln_cols_kernel, dim3((2 * cols + 15) / 16), dim3(1024), 0, (hipStream_t)stream, (const float*)ws,
                       rows > 0 ? s.grid : 0, cols, dgamma, dbeta, accumulate);
    MMST_CHECK_LAUNCH();
  }
  return MMST_OK;
}

}  // extern "C"
