// Linear layer with softmax cross entropy over a large vocabulary, loss and gradients, without the logits in memory.
//
//   l[n][v] = sum_d h[n][d] w[v][d] + bias[v]          lse[n] = log sum_v exp l[n][v]       loss[n] = lse[n] - l[n][t_n]
//   g[n][v] = dloss[n] (exp(l[n][v] - lse[n]) - [v == t_n])        dh = g w        dw = g^T h        dbias = sum_n g
//
// All of it is matrix products over tiles of 256 x 256 (or 128 x 128, see large_tiles) on v_mfma_f32_16x16x32_bf16 with
// fp32 accumulation; the softmax is made from the tile's logits while they are in registers:
//   logits a tile becomes (max, sum exp) per row and 64 words, 8 bytes; for the gradient also its exponentials, 16 bits
//   rows   a row's pairs are joined into lse and the loss
//   scale  the exponentials become g, in place
//   dh, dw products with g, whose operands lie along the wrong axis and are read through transposing LDS reads
// Three products, then, where computing the logits twice would take four; the price is one more rounding of a probability
// (pack_exp, 2^-10 of itself) and one pass over g.  With a short contraction the pass would cost more than the product:
// those layers compute the logits twice (ce_stream_kernel).
// The gradient goes in pieces of the ROWS: a piece's g [rows][V] is the only large buffer.  Rows that do not count
// (ignore_index) are left out at the start: the others are numbered through on the device and gathered, so a padded batch
// costs what its tokens cost, and what padding holds (NaN, infinities) reaches nothing.  The loss alone does that where it
// pays (numbers), and otherwise drops the results of such rows, which reach no other row.
// g is made for weights relative to the largest one, which the products' results are multiplied with in fp32: weights that are
// all the same (a mean's 1 / rows) are 1 then, and g of a target, near -1 in most rows, is near -1 in bf16 as well.  Rounded with
// 1 / rows inside, all of them would be off by the same 2^-8 at worst, and so would their sum.
#include "../../include/mmst.h"
#include "common.h"

namespace {

typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef LDS_AS unsigned char lds_byte;
typedef __attribute__((address_space(3))) void* lptr_t;
constexpr float LOG2E = 1.4426950408889634f;
// exp(x - m) is one fused multiply-add, exp2(x log2 e - m log2 e), and one exponential; the rounding of m log2 e costs digits
// where m is large (and everything where it is a mask's -1e30), so beyond this the difference is taken first.
constexpr float FAR = 4096.f;
constexpr int VT = 256;   // g is padded to whole tiles of the vocabulary, its rows to whole tiles as well

// Exponentials on their way to g, two in 32 bits.  They lie in [0, 2), so neither the sign nor the top bit of a float's exponent
// says anything: bits 29..14 are 7 of the exponent and 9 of the mantissa, two more than bf16 keeps.  They are rounded by 2^-10
// here and by 2^-8 as g, all but as if g had been rounded alone; in bf16 the errors of dbias were 1.4 times as large.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint32_t pack_exp(float lo, float hi) {
  const uint32_t a = (__builtin_bit_cast(uint32_t, lo) << 2) + 0x8000u, b = (__builtin_bit_cast(uint32_t, hi) << 2) + 0x8000u;
  return __builtin_amdgcn_perm(b, a, 0x07060302);   // the upper halves
}
__device__ __forceinline__ float unpack_exp(uint32_t w, int upper) {
  return __builtin_bit_cast(float, (upper ? w >> 2 : w << 14) & 0x3FFFC000u);
}

enum { LOGIT_STATS = 0, LOGIT_GRAD = 1, DH = 2, DW = 3, LOGIT_EXP = 4, LOGIT_LOSS = 5, LOGIT_PART = 6 };

struct CeGemm {
  const bf16* P; const bf16* Q;      // operands; the token / vocabulary side of the output's rows, and its columns
  long ldp, ldq;
  int Pn, Qn, K;                     // extents; K for DH is the vocabulary
  const int* count;                  // device: rows that count; the piece holds clamp(count - row0, 0, rows_max) of them
  int row0, rows_max;                // (count == NULL: rows_max rows)
  int ptiles, qtiles, ksplit;        // ksplit: parts of the contraction
  // logits
  const float* bias; const int64_t* target; const int* index;
  const int* word;                   // the targets of the rows that count (gradient; NULL: target[row])
  float2* part; float* tlogit;       // per 64 words and row: max, sum of exp; the target's logit
  const float2* lse;                 // the row's maximum, and log2 of its sum of exponentials
  const float* weight;               // of the rows' losses in g, relative to *unit
  const float* unit; bf16* g; long ldg;
  float* loss_out; float* lse_out; int64_t ignore;   // LOGIT_LOSS; joining scale
  // products
  void* out; long ldo; int out_f32;                   // out_f32: fp32, else bf16
  const float* acc_in; float* slab; float* slab_bias;   // slabs: [ksplit][Pn][ldslab], [ksplit][Pn]
  int ldslab;
  void* dbias; const float* dbias_in; int dbias_f32;  // DW: sums of g over the rows; added to dbias_in
};

__device__ __forceinline__ int piece_rows(const CeGemm& a) {
  if (!a.count) return a.rows_max;
  const int left = *a.count - a.row0;
  return left < 0 ? 0 : left < a.rows_max ? left : a.rows_max;
}

// One operand's tile in LDS: B rows (or columns) x BK of the contraction.
//   rows along the contraction (T == false): B rows of 2 BK bytes, the 16-byte pieces of a row exchanged by its key
//   columns along the contraction (T == true): BK rows of 2 B bytes, their 32-byte pieces exchanged by the row's key
// The exchange makes the fragment reads of 16 rows hit all banks; it is applied to the SOURCE address, since the LDS-DMA
// writes lane i's 16 bytes at i * 16.  What lies outside the operand reads as zero (the buffer's bounds check; the tail of
// the contraction by an offset past every bound).
template <bool T, bool QSIDE, int B, int NTHR, int BK> struct Operand {
  static constexpr int PIECES = B * BK / 8, NI = PIECES / NTHR;   // 16-byte pieces; DMA instructions per thread and step
  static constexpr int BYTES = B * BK * 2, ROW = BK / 8;          // pieces per row (!T)
  static constexpr uint32_t OUT = 0xFFFFFFF0u;
  static_assert(PIECES % NTHR == 0 && BK == 64, "tile shape");
  uint32_t off[NI];
  const bf16* base;
  long ld;
  int K, wide;   // wide: columns of the operand right of the tile's first (T)
  long rows;     // rows of the operand below the tile's first (!T)

  // a fragment reads 16 rows: r0 + i (P), r0 + 8 (i >> 2) + 4 half + (i & 3) (Q); 64 banks of 4 bytes
  static __device__ __forceinline__ int key(int r) {
    if constexpr (T) return (r & 3) | (((r >> 3) & 1) << 2);
    else return QSIDE ? (r & 3) | (((r >> 3) & 1) << 2) : r & 7;
  }
  static __device__ __forceinline__ int piece(int slot) { const int r = slot / ROW; return (slot % ROW) ^ key(r); }   // (!T)

  __device__ __forceinline__ void seek(const bf16* p, int first, int n) {   // another tile of the operand
    base = T ? p + first : p + (long)first * ld;
    rows = wide = n - first;
  }
  __device__ __forceinline__ void init(const bf16* p, long ld_, int first, int n, int K_, int tid) {
    ld = ld_;
    K = K_;
    seek(p, first, n);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int slot = i * NTHR + tid;
      if constexpr (!T) {
        off[i] = (uint32_t)((slot / ROW) * (int)ld_ * 2 + piece(slot) * 16);
      } else {
        const int r = slot / (B / 8), c16 = slot % (B / 8);
        off[i] = (uint32_t)(r * (int)ld_ * 2 + ((((c16 >> 1) ^ key(r)) << 1) | (c16 & 1)) * 16);
      }
    }
  }
  // DMA instructions lo .. hi - 1 of step k0
  template <int LO, int HI> __device__ __forceinline__ void issue(lds_byte* img, int k0, int tid, int wave) const {
    const bf16* p;
    long bytes;
    if constexpr (!T) {
      p = base + k0;
      bytes = ((rows - 1) * ld + ((K + 7) & ~7) - k0) * 2;   // whole 16-byte pieces: g's rows are padded
    } else {
      p = base + (long)k0 * ld;
      bytes = ((long)(K - k0 - 1) * ld + ((wide + 7) & ~7)) * 2;
    }
    bytes = bytes < 0 ? 0 : bytes > 0x7FFFFFFF ? 0x7FFFFFFF : bytes;
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)bytes, 0x00020000);
    const bool tail = !T && K - k0 < BK;   // of the contraction (uniform)
#pragma unroll
    for (int i = LO; i < HI; ++i) {
      uint32_t o = off[i];
      if (tail) o = piece(i * NTHR + tid) * 8 >= K - k0 ? OUT : o;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lptr_t)(img + i * NTHR * 16 + wave * 1024), 16, (int)o, 0, 0, 0);
    }
  }
  // fragment of 16 rows at r0 for the 32 contraction steps ks: lane (i = lane & 15, j = lane >> 4) gets row i, steps 8 j ..
  // 8 j + 7.  QSIDE: two fragments (half 0, 1) leave eight consecutive columns of the result in a lane.
  __device__ __forceinline__ static bf16x8 frag(const lds_byte* img, int r0, int half, int ks, int lane) {
    if constexpr (!T) {
      const int i = lane & 15;
      const int r = QSIDE ? r0 + 8 * (i >> 2) + 4 * half + (i & 3) : r0 + i;
      const int c = (ks * 4 + (lane >> 4)) ^ key(r);
      return *reinterpret_cast<const LDS_AS bf16x8*>(img + r * (BK * 2) + c * 16);
    } else {
      const int k = ks * 32 + 8 * (lane >> 4) + ((lane & 15) >> 2);
      const int col = QSIDE ? r0 + 8 * (lane & 3) + 4 * half : r0 + 4 * (lane & 3);
      const lds_byte* p = img + k * (B * 2) + (((col >> 4) ^ key(k)) << 5) + (col & 15) * 2;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS s16x4*)p);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS s16x4*)(p + 4 * (B * 2)));   // (same key)
      return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
};

template <int MODE, int BP, int BQ, int WP, int WQ, int STAGES = 2>
struct CeTile {
  static constexpr int NW = WP * WQ, NTHR = NW * 64, MT = BP / WP / 16, NT = BQ / WQ / 16;
  static constexpr bool TP = MODE == DW, TQ = MODE == DH || MODE == DW;
  static constexpr int BK = 64, NS = STAGES;   // a step of the contraction; stages of LDS
  using OpP = Operand<TP, false, BP, NTHR, BK>;
  using OpQ = Operand<TQ, true, BQ, NTHR, BK>;
  static constexpr int STAGE = OpP::BYTES + OpQ::BYTES, SMEM = NS * STAGE;

  struct Frags { bf16x8 p[MT], q[NT]; };
  // SUM (DW): also the sums of the P operand over the contraction, as one more product against ones
  template <bool SUM> struct Acc {
    f32x4 v[MT][NT];
    f32x4 sum[SUM ? MT : 1];
    __device__ __forceinline__ void clear() {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) v[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < (SUM ? MT : 1); ++i) sum[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    __device__ __forceinline__ void add(const Frags& f, int mt) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) v[mt][nt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.q[nt], f.p[mt], v[mt][nt], 0, 0, 0);
      if constexpr (SUM) {
        bf16x8 ones;
#pragma unroll
        for (int e = 0; e < 8; ++e) ones[e] = (bf16)1.0f;
        sum[mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, f.p[mt], sum[mt], 0, 0, 0);
      }
    }
  };
  static __device__ __forceinline__ void read(Frags& f, const lds_byte* rd, int ks, int pw0, int qw0, int lane) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) f.q[nt] = OpQ::frag(rd + OpP::BYTES, qw0 + (nt >> 1) * 32, nt & 1, ks, lane);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) f.p[mt] = OpP::frag(rd, pw0 + mt * 16, 0, ks, lane);
  }
  // DMA instructions LO .. HI - 1 of the step's PER: the P operand's, then the Q operand's
  static constexpr int PER = OpP::NI + OpQ::NI;
  template <int LO, int HI>
  static __device__ __forceinline__ void issue(const OpP& p, const OpQ& q, lds_byte* wr, int k, int tid, int wave) {
    if constexpr (LO < OpP::NI) p.template issue<LO, (HI < OpP::NI ? HI : OpP::NI)>(wr, k, tid, wave);
    if constexpr (HI > OpP::NI) q.template issue<(LO > OpP::NI ? LO - OpP::NI : 0), HI - OpP::NI>(wr + OpP::BYTES, k, tid, wave);
  }

  // One step: the next step's operands are requested into `wr`, the products of `rd` are made.  The two never
  // overlap, and saying so is what keeps the compiler from waiting for the DMA before every LDS read.
  template <bool SUM>
  static __device__ __forceinline__ void step(Acc<SUM>& acc, const OpP& p, const OpQ& q, lds_byte* __restrict__ wr,
                                              const lds_byte* __restrict__ rd, bool more, int k1, int tid, int wave,
                                              int pw0, int qw0, int lane) {
    if (more) issue<0, PER>(p, q, wr, k1, tid, wave);
#pragma unroll
    for (int ks = 0; ks < BK / 32; ++ks) {
      Frags f;
      read(f, rd, ks, pw0, qw0, lane);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) acc.add(f, mt);
    }
  }

  // Eight waves in two halves, one of each on every SIMD: while one half reads the fragments of 32 contraction steps, the
  // other multiplies, and a barrier changes the roles.  Phases of step s, each ended by a barrier of the whole workgroup:
  //              4 s                4 s + 1        4 s + 2       4 s + 3
  //   first      read 0             multiply 0     read 1        multiply 1
  //   second     multiply 1 (s-1)   read 0         multiply 0    read 1
  // The stage of step s - 1 is free at phase 4 s; the DMA of step s + NS - 1 goes there in phases 4 s and 4 s + 1, half of
  // it each, behind the reads or between the products: issued in one go it would hold up whichever comes after it, since
  // the address unit takes 18 cycles for each of the 64 instructions.  Step s + 1 is waited for before the last barrier of s.
  static __device__ __forceinline__ void fence() { __builtin_amdgcn_sched_barrier(0); }
  static __device__ __forceinline__ void barrier() { asm volatile("s_barrier" ::: "memory"); fence(); }
  static __device__ __forceinline__ void reads_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
  static __device__ __forceinline__ void dma_done() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 2) * PER) : "memory"); }
  static __device__ __forceinline__ void all_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
  template <bool SUM> static __device__ __forceinline__ void multiply(Acc<SUM>& acc, const Frags& f) {
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) acc.add(f, mt);
    __builtin_amdgcn_s_setprio(0);
    fence();
  }
  // the products with DMA instructions LO .. LO + PER / 2 - 1 between them, evenly
  template <int LO, int MT0 = 0, bool SUM>
  static __device__ __forceinline__ void multiply_issue(Acc<SUM>& acc, const Frags& f, const OpP& p, const OpQ& q, lds_byte* wr,
                                                        int k, int tid, int wave) {
    constexpr int N = PER / 2;
    if constexpr (MT0 == 0) __builtin_amdgcn_s_setprio(1);
    acc.add(f, MT0);
    fence();
    constexpr int lo = MT0 * N / MT, hi = (MT0 + 1) * N / MT;
    if constexpr (hi > lo) {
      issue<LO + lo, LO + hi>(p, q, wr, k, tid, wave);
      fence();
    }
    if constexpr (MT0 + 1 < MT) multiply_issue<LO, MT0 + 1>(acc, f, p, q, wr, k, tid, wave);
    else __builtin_amdgcn_s_setprio(0);
  }
  template <bool SUM>
  static __device__ __forceinline__ void step_first(Acc<SUM>& acc, const OpP& p, const OpQ& q, lds_byte* __restrict__ wr,
                                                    const lds_byte* __restrict__ rd, int k1, int tid, int wave, int pw0,
                                                    int qw0, int lane) {
    Frags f;
    read(f, rd, 0, pw0, qw0, lane);
    fence();
    issue<0, PER / 2>(p, q, wr, k1, tid, wave);
    reads_done();
    barrier();
    multiply_issue<PER / 2>(acc, f, p, q, wr, k1, tid, wave);
    barrier();
    read(f, rd, 1, pw0, qw0, lane);
    reads_done();
    barrier();
    multiply(acc, f);
    dma_done();
    barrier();
  }
  template <bool SUM>
  static __device__ __forceinline__ void step_second(Acc<SUM>& acc, Frags& f, const OpP& p, const OpQ& q,
                                                     lds_byte* __restrict__ wr, const lds_byte* __restrict__ rd, int k1,
                                                     int tid, int wave, int pw0, int qw0, int lane) {
    multiply_issue<0>(acc, f, p, q, wr, k1, tid, wave);
    barrier();
    read(f, rd, 0, pw0, qw0, lane);
    fence();
    issue<PER / 2, PER>(p, q, wr, k1, tid, wave);
    reads_done();
    barrier();
    multiply(acc, f);
    barrier();
    read(f, rd, 1, pw0, qw0, lane);
    reads_done();
    dma_done();
    barrier();
  }

  // A tile's products: prime() requests its first NS - 1 steps (nobody may be reading a stage), ready() waits for the first,
  // steps() makes them all.  There is no branch inside a step: the last ones request steps that are not there, which move
  // nothing but zeros (or, in a split contraction, the next part's first steps) into stages that nobody reads, and the second
  // half starts by multiplying zeros.  Behind steps() nobody reads a stage.
  static __device__ __forceinline__ void prime(const OpP& p, const OpQ& q, lds_byte* lds, int kbeg, int tid, int wave) {
    all_done();
#pragma unroll
    for (int s = 0; s < NS - 1; ++s) issue<0, PER>(p, q, lds + s * STAGE, kbeg + s * BK, tid, wave);
  }
  static __device__ __forceinline__ void ready() {
    dma_done();
    barrier();
  }
  template <bool SUM>
  static __device__ __forceinline__ void steps(Acc<SUM>& acc, const OpP& p, const OpQ& q, lds_byte* lds, int kbeg, int nsteps,
                                               int tid, int wave, int pw0, int qw0, int lane) {
    if constexpr (NW != 8) {
      int rd = 0, wr = NS - 1;
      for (int s = 0; s < nsteps; ++s) {
        // this wave's share of step s has landed and its reads of step s - 1 are done; behind the barrier everybody's have, and
        // nobody reads the stage of step s - 1
        if (s) {
          reads_done();
          dma_done();
          asm volatile("s_barrier" ::: "memory");
        }
        // (two stages: nothing is requested behind the last step; more: always, so that what is in flight can be counted)
        step(acc, p, q, lds + wr * STAGE, lds + rd * STAGE, NS > 2 || s + 1 < nsteps, kbeg + (s + NS - 1) * BK, tid, wave, pw0,
             qw0, lane);
        wr = rd;
        rd = rd + 1 == NS ? 0 : rd + 1;
      }
      reads_done();
      if constexpr (NS > 2) all_done();
      barrier();
    } else {
      int rd = 0, wr = NS - 1;
      if (wave < 4) {
        for (int s = 0; s < nsteps; ++s) {
          step_first(acc, p, q, lds + wr * STAGE, lds + rd * STAGE, kbeg + (s + NS - 1) * BK, tid, wave, pw0, qw0, lane);
          wr = rd;
          rd = rd + 1 == NS ? 0 : rd + 1;
        }
        barrier();   // the second half's last multiplication
      } else {
        Frags f = {};
        for (int s = 0; s < nsteps; ++s) {
          step_second(acc, f, p, q, lds + wr * STAGE, lds + rd * STAGE, kbeg + (s + NS - 1) * BK, tid, wave, pw0, qw0, lane);
          wr = rd;
          rd = rd + 1 == NS ? 0 : rd + 1;
        }
        multiply(acc, f);
        barrier();
      }
    }
  }
};

// consecutive tiles in groups of eight rows of tiles: what runs at the same time on one XCD shares its operands in the L2
__device__ __forceinline__ void tile_of(int id, int ptiles, int qtiles, int& pt, int& qt) {
  const int group = 8 * qtiles, gi = id / group, gp = ptiles - gi * 8 < 8 ? ptiles - gi * 8 : 8;
  const int in = id - gi * group;
  pt = gi * 8 + in % gp;
  qt = in / gp;
}

// ---------------------------------------------------------------------------------------------------- products with g
// dh of a piece or dw, one tile per workgroup.  The matrix units work in 0.63 (dh) and 0.69 (dw) of the cycles, at the 1.6 to 1.8
// GHz that the card's power leaves; 8192 x 2048 x 65536 takes 1.81 ms for dh and 1.76 ms for dw, 1.21 and 1.25 PFLOP/s in 256 x
// 256 tiles (2.15 and 2.2 ms with
// four waves of 128 x 128 each, that issue their DMA, read and multiply one after another).  In narrow layers by reading g: 3032
// x 128 x 32000 takes 66 us for both, 388 MB at 5.9 TB/s.
// block: the workgroup's number of n
template <int MODE, int BP, int BQ, int WP, int WQ, int STAGES = 2>
__device__ __forceinline__ void ce_product(const CeGemm& a, int block, int n, lds_byte* lds) {
  using Tile = CeTile<MODE, BP, BQ, WP, WQ, STAGES>;
  constexpr int MT = Tile::MT, NT = Tile::NT;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int id;   // consecutive tiles to one XCD (workgroups go round the eight of them)
  {
    const int q8 = n >> 3, r8 = n & 7, x = block & 7;
    id = (x < r8 ? x * (q8 + 1) : r8 * (q8 + 1) + (x - r8) * q8) + (block >> 3);
  }
  const int per = a.ptiles * a.qtiles;
  const int ks_id = id / per;
  if (ks_id >= a.ksplit) return;   // (uniform, as the next)
  id -= ks_id * per;
  int pt, qt;
  tile_of(id, a.ptiles, a.qtiles, pt, qt);
  const int rows = piece_rows(a);
  const int p0 = pt * BP, q0 = qt * BQ;
  const int K = MODE == DW ? rows : a.K, Pn = MODE == DW ? a.Pn : rows;
  if (MODE != DW && p0 >= rows) return;
  int kbeg = 0, nsteps = (K + Tile::BK - 1) / Tile::BK;
  if (a.ksplit > 1) {
    const int s0 = (int)((long)nsteps * ks_id / a.ksplit), s1 = (int)((long)nsteps * (ks_id + 1) / a.ksplit);
    kbeg = s0 * Tile::BK;
    nsteps = s1 - s0;
  }
  const int pw0 = (wave / WQ) * (BP / WP), qw0 = (wave % WQ) * (BQ / WQ);
  typename Tile::OpP op;
  typename Tile::OpQ oq;
  op.init(a.P, a.ldp, p0, Pn, K, tid);
  oq.init(a.Q, a.ldq, q0, a.Qn, K, tid);

  typename Tile::template Acc<false> plain;
  f32x4 (&acc)[MT][NT] = plain.v;
  if (nsteps > 0) {
    Tile::prime(op, oq, lds, kbeg, tid, wave);
    Tile::ready();
  }
  if (MODE == DW && a.dbias && qt == 0 && wave % WQ == 0) {   // the waves that also have the sums over the rows
    typename Tile::template Acc<MODE == DW> sums;
    sums.clear();
    Tile::steps(sums, op, oq, lds, kbeg, nsteps, tid, wave, pw0, qw0, lane);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int v = p0 + pw0 + mt * 16 + (lane & 15);
      if (lane < 16 && v < Pn) {
        const float x = sums.sum[MODE == DW ? mt : 0][0] * (a.slab ? 1.f : *a.unit) + (a.dbias_in && !a.slab ? a.dbias_in[v] : 0.f);
        if (a.slab) a.slab_bias[(size_t)ks_id * Pn + v] = x;
        else if (a.dbias_f32) ((float*)a.dbias)[v] = x;
        else ((bf16*)a.dbias)[v] = (bf16)x;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) acc[mt][nt] = sums.v[mt][nt];
    }
  } else {
    plain.clear();
    Tile::steps(plain, op, oq, lds, kbeg, nsteps, tid, wave, pw0, qw0, lane);
  }

  const int i16 = lane & 15, j4 = lane >> 4;
  const float unit = a.slab ? 1.f : *a.unit;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int m = p0 + pw0 + mt * 16 + i16;
    if (m >= Pn) continue;
#pragma unroll
    for (int tp = 0; tp < NT / 2; ++tp) {
      const int c = q0 + qw0 + tp * 32 + 8 * j4;
      if (c >= a.Qn) continue;   // (Qn is a multiple of 8, or the slabs' rows are padded to one)
      f32x4 lo = acc[mt][2 * tp] * unit, hi = acc[mt][2 * tp + 1] * unit;
      if (a.slab) {
        float* d = a.slab + ((size_t)ks_id * a.Pn + m) * a.ldslab + c;
        *reinterpret_cast<f32x4*>(d) = lo;
        *reinterpret_cast<f32x4*>(d + 4) = hi;
        continue;
      }
      const size_t row = MODE == DH ? (size_t)a.index[m] : (size_t)m;
      if (MODE == DW && a.acc_in) {
        const float* s = a.acc_in + row * a.Qn + c;
        lo += *reinterpret_cast<const f32x4*>(s);
        hi += *reinterpret_cast<const f32x4*>(s + 4);
      }
      if (MODE == DW && a.out_f32) {
        float* d = (float*)a.out + row * a.ldo + c;
        *reinterpret_cast<f32x4*>(d) = lo;
        *reinterpret_cast<f32x4*>(d + 4) = hi;
      } else {
        bf16x8 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) { o[e] = (bf16)lo[e]; o[4 + e] = (bf16)hi[e]; }
        *reinterpret_cast<bf16x8*>((bf16*)a.out + row * a.ldo + c) = o;
      }
    }
  }
}

template <int MODE, int BP, int BQ, int WP, int WQ, int STAGES = 2>
__global__ __launch_bounds__(WP * WQ * 64, WP * WQ * 64 == 512 ? 2 : 1) void ce_product_kernel(const CeGemm a) {
  __shared__ __attribute__((aligned(1024))) unsigned char smem[CeTile<MODE, BP, BQ, WP, WQ, STAGES>::SMEM];
  ce_product<MODE, BP, BQ, WP, WQ, STAGES>(a, blockIdx.x, gridDim.x, (lds_byte*)smem);
}

// Both products in one launch, where both have small tiles: n workgroups (a multiple of 8, so that the others' XCDs are what
// their numbers say) for dh, the others for dw.  All of the gradient of 4032 x 128 x 43: 42 us with a launch each and 36 with
// one; of 2000 x 128 x 8000: 80 and 65; of 3032 x 128 x 32000: 203 and, with parts for 256 workgroups of each, 167.
__global__ __launch_bounds__(256, 1) void ce_products_kernel(const CeGemm dh, const CeGemm dw, int n) {
  __shared__ __attribute__((aligned(1024))) unsigned char smem[CeTile<DW, 128, 128, 2, 2>::SMEM];
  if ((int)blockIdx.x < n) ce_product<DH, 128, 128, 2, 2>(dh, blockIdx.x, n, (lds_byte*)smem);
  else ce_product<DW, 128, 128, 2, 2>(dw, (int)blockIdx.x - n, (int)gridDim.x - n, (lds_byte*)smem);
}

// ---------------------------------------------------------------------------------------------------- logits, tile by tile
// A workgroup walks over tiles of the logits (one workgroup per CU with large tiles, two with small ones); the first steps of
// the next tile's contraction are requested before this tile's softmax, which a wave does for its 64 columns (or 160) alone.
// LOGIT_STATS: (max, sum of exponentials) per row and 64 words (160).  LOGIT_EXP: these, and the exponentials themselves.  8192 x
// 2048 x 65536: 2.02 ms with the exponentials, 1.09 PFLOP/s; the matrix units work in 0.56 of the cycles, and nothing multiplies
// beside the softmax at the ends of the tiles.  333 x 1024 x 50001: 45 us in two rounds of 128 x 160 (matrix units 0.42), 50 in
// three of 128 x 128.
template <int MODE, int BP, int BQ, int WP, int WQ, int STAGES = 2>
__global__ __launch_bounds__(WP * WQ * 64, STAGES == 2 ? 2 : 1) void ce_logits_kernel(const CeGemm a) {
  using Tile = CeTile<MODE, BP, BQ, WP, WQ, STAGES>;
  constexpr int MT = Tile::MT, NT = Tile::NT;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[Tile::SMEM];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rows = piece_rows(a);
  const int ptiles = (rows + BP - 1) / BP, tiles = ptiles * a.qtiles;
  // an XCD (workgroups go round the eight of them) has a run of consecutive tiles, its workgroups take them in turn
  const int xcd = blockIdx.x & 7, group = (int)gridDim.x >> 3, chunk = (tiles + 7) >> 3;
  const int end = (xcd + 1) * chunk < tiles ? (xcd + 1) * chunk : tiles;
  int id = xcd * chunk + ((int)blockIdx.x >> 3);
  if (id >= end) return;   // (uniform)
  const int pw0 = (wave / WQ) * (BP / WP), qw0 = (wave % WQ) * (BQ / WQ);
  const int i16 = lane & 15, j4 = lane >> 4;
  const int nsteps = (a.K + Tile::BK - 1) / Tile::BK;
  lds_byte* const lds = (lds_byte*)smem;
  const __amdgpu_buffer_rsrc_t bias_rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)a.bias, 0, a.bias ? a.Qn * 4 : 0, 0x00020000);

  int pt, qt;
  tile_of(id, ptiles, a.qtiles, pt, qt);
  typename Tile::OpP op;
  typename Tile::OpQ oq;
  op.init(a.P, a.ldp, pt * BP, rows, a.K, tid);
  oq.init(a.Q, a.ldq, qt * BQ, a.Qn, a.K, tid);
  Tile::prime(op, oq, lds, 0, tid, wave);
  for (;;) {
    const int p0 = pt * BP, q0 = qt * BQ;
    Tile::ready();
    // bias (0 past the vocabulary and without one) and targets, there when the products are
    float raw[NT / 2][8];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int at = (q0 + qw0 + 8 * j4) * 4 + (i >> 1) * 128 + (i & 1) * 16;
      const f32x4 v = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(bias_rsrc, at, 0, 0));
#pragma unroll
      for (int e = 0; e < 4; ++e) raw[i >> 1][(i & 1) * 4 + e] = v[e];
    }
    int target[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      int m = p0 + pw0 + mt * 16 + i16;
      m = m < rows ? m : rows - 1;
      target[mt] = a.word ? a.word[m] : (int)(a.target[m] >= 0 && a.target[m] < a.Qn ? a.target[m] : -1 << 30);
    }
    typename Tile::template Acc<false> plain;
    f32x4 (&acc)[MT][NT] = plain.v;
    plain.clear();
    Tile::steps(plain, op, oq, lds, 0, nsteps, tid, wave, pw0, qw0, lane);

    const int next = id + group;
    int pt1 = pt, qt1 = qt;
    if (next < end) {
      tile_of(next, ptiles, a.qtiles, pt1, qt1);
      op.seek(a.P, pt1 * BP, rows);
      oq.seek(a.Q, qt1 * BQ, a.Qn);
      Tile::prime(op, oq, lds, 0, tid, wave);
    }

    // logits: row i16 of each 16, columns 32 tp + 8 j4 + e
    const bool edge = q0 + BQ > a.Qn;
#pragma unroll
    for (int tp = 0; tp < NT / 2; ++tp)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float b = raw[tp][e];
        if (edge && q0 + qw0 + tp * 32 + 8 * j4 + e >= a.Qn) b = -INFINITY;   // past the vocabulary
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) acc[mt][2 * tp + (e >> 2)][e & 3] += b;
      }
    const int base = q0 + qw0 + 8 * j4;
    auto mine = [&](int word) { return (unsigned)(word - base) < NT * 16u && ((word - base) & 24) == 0; };   // 32 tp + 0..7
    bool any = false;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) any |= mine(target[mt]);
    const bool targets = __ballot(any) != 0;
    float mx[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float v = acc[mt][0][0];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) v = fmaxf(v, acc[mt][nt][e]);
      mx[mt] = xor32_max(xor16_max(v));
      if (targets) {
        const int m = p0 + pw0 + mt * 16 + i16;
        float x = 0.f;
#pragma unroll
        for (int tp = 0; tp < NT / 2; ++tp)
#pragma unroll
          for (int e = 0; e < 8; ++e) x = target[mt] - base == tp * 32 + e ? acc[mt][2 * tp + (e >> 2)][e & 3] : x;
        if (mine(target[mt]) && m < rows) a.tlogit[m] = x;
      }
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float at = mx[mt] == -INFINITY ? 0.f : mx[mt];   // nothing but masked words: exp(-inf - 0), not of NaN
      if (__ballot(fabsf(at) > FAR)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[mt][nt][e] -= at;
        at = 0.f;
      }
      at *= LOG2E;
      float x = 0.f;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          acc[mt][nt][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[mt][nt][e], LOG2E, -at));
          x += acc[mt][nt][e];
        }
      x = xor32_sum(xor16_sum(x));
      const int m = p0 + pw0 + mt * 16 + i16;
      if (j4 == 0 && m < rows) a.part[(size_t)(qt * WQ + wave % WQ) * a.rows_max + m] = make_float2(mx[mt], x);
    }
    if constexpr (MODE == LOGIT_EXP) {   // whole tiles: g has rows and columns for them
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int tp = 0; tp < NT / 2; ++tp) {
          u32x4 o;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const f32x4& x = acc[mt][2 * tp + (e >> 1)];
            o[e] = pack_exp(x[(2 * e) & 3], x[(2 * e + 1) & 3]);
          }
          *reinterpret_cast<u32x4*>(a.g + (size_t)(p0 + pw0 + mt * 16 + i16) * a.ldg + q0 + qw0 + tp * 32 + 8 * j4) = o;
        }
    }
    if (next >= end) return;
    id = next;
    pt = pt1;
    qt = qt1;
  }
}

// Logits in parts of their contraction (LOGIT_PART: slabs, as of the other split products), for layers so wide and tiles so few
// that the steps of one tile are what takes the time.  This joins them: 16 rows x 64 words per workgroup, four words per lane,
// and leaves what the tiles leave otherwise.
template <int MODE> __global__ __launch_bounds__(256) void ce_join_kernel(const CeGemm a) {
  const int rows = piece_rows(a), m = blockIdx.y * 16 + (threadIdx.x >> 4), c = blockIdx.x * 64 + (threadIdx.x & 15) * 4;
  if ((int)blockIdx.y * 16 >= rows) return;
  const int r = m < rows ? m : rows - 1;
  f32x4 x = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  if (c < a.Qn) {
    const float* p = a.slab + (size_t)r * a.ldslab + c;
    const size_t stride = (size_t)a.Pn * a.ldslab;
    x = *reinterpret_cast<const f32x4*>(p);
#pragma unroll 4
    for (int k = 1; k < a.ksplit; ++k) x += *reinterpret_cast<const f32x4*>(p + k * stride);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (c + e >= a.Qn) x[e] = -INFINITY;
    else if (a.bias) x[e] += a.bias[c + e];
  }
  const int64_t t = a.word ? a.word[r] : a.target[r];
  if (t >= c && t < c + 4 && t < a.Qn && m < rows) a.tlogit[m] = t == c ? x[0] : t == c + 1 ? x[1] : t == c + 2 ? x[2] : x[3];
  const float mx = row16_max(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]))), at = mx == -INFINITY ? 0.f : mx;
  float sum = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[e] = __builtin_amdgcn_exp2f((x[e] - at) * LOG2E);
    sum += x[e];
  }
  sum = row16_sum(sum);
  if (m >= rows) return;
  if ((threadIdx.x & 15) == 0) a.part[(size_t)blockIdx.x * a.rows_max + m] = make_float2(mx, sum);
  if constexpr (MODE == LOGIT_EXP) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    *reinterpret_cast<u32x2*>(a.g + (size_t)m * a.ldg + c) = u32x2{pack_exp(x[0], x[1]), pack_exp(x[2], x[3])};
  }
}

// g from the exponentials of a piece, in place: a tile's times exp(its maximum - the row's lse) and the weight; of the target's
// word from its logit, which is there in fp32.  Four rows per workgroup and 2048 columns, 16 bytes per lane; bound by HBM: 2.1
// GB in 0.41 ms, 5.2 TB/s.
// JOIN: a wave first joins the pairs of one of the rows, which saves the launch of ce_rows_kernel; every 2048 columns do that
// again, so only up to JOIN_VOCAB words.  All of the gradient, joined here / apart: 4032 x 128 x 43 35 / 37 us, 700 x 136 x 5000
// 44 / 47, 1000 x 128 x 8000 49 / 54, 2000 x 136 x 16000 107 / 106, 1000 x 256 x 32000 121 / 114.
template <bool JOIN> __global__ __launch_bounds__(256) void ce_scale_kernel(const CeGemm a, int pairs) {
  __shared__ float2 joined[4];
  const int rows = piece_rows(a), across = (int)((a.ldg + 2047) / 2048), r0 = (int)(blockIdx.x / across) * 4;
  const int c = (int)(blockIdx.x % across) * 2048 + (int)threadIdx.x * 8;
  if (r0 >= rows) return;   // (uniform)
  if constexpr (JOIN) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r = r0 + w;
    if (r < rows) {
      float m = -INFINITY, s = 0.f;
      for (int q = lane; q < pairs; q += 64) {
        const float2 p = a.part[(size_t)q * a.rows_max + r];
        const float top = fmaxf(m, p.x), at = top == -INFINITY ? 0.f : top;
        s = s * __builtin_amdgcn_exp2f((m - at) * LOG2E) + p.y * __builtin_amdgcn_exp2f((p.x - at) * LOG2E);
        m = top;
      }
      const float top = wave_max(m), at = top == -INFINITY ? 0.f : top;
      s = wave_sum(s * __builtin_amdgcn_exp2f((m - at) * LOG2E));
      if (lane == 0) {
        joined[w] = make_float2(top, log2f(s));
        if (blockIdx.x % across == 0) {
          const int n = a.index[r];
          const float ls = logf(s), l = at + ls;
          a.loss_out[n] = l == -INFINITY ? INFINITY : ls + (at - a.tlogit[r]);
          if (a.lse_out) a.lse_out[n] = l;
        }
      }
    }
    __syncthreads();
  }
  if (c >= a.Qn) return;
  u32x4 x[4];
  float scale[4], wt[4], gt[4];   // gt: g of the target's word, whose 1 would leave an exponential's last digits
  int hit[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + i < rows ? r0 + i : rows - 1;
    x[i] = *reinterpret_cast<const u32x4*>(a.g + (size_t)r * a.ldg + c);
    const float2 l = JOIN ? joined[r - r0] : a.lse[r];
    wt[i] = a.weight[r];
    hit[i] = a.word[r] - c;
    // a row whose every logit is masked has no gradient
    if (l.y == -INFINITY) wt[i] = 0.f;
    const float top = a.part[(size_t)(c / 64) * a.rows_max + r].x;
    gt[i] = l.y == -INFINITY ? 0.f : (__builtin_amdgcn_exp2f((a.tlogit[r] - l.x) * LOG2E - l.y) - 1.f) * wt[i];
    scale[i] = l.y == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((top - l.x) * LOG2E - l.y) * wt[i];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (r0 + i >= rows) break;
    bf16x8 o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = (bf16)(hit[i] == e ? gt[i] : unpack_exp(x[i][e >> 1], e & 1) * scale[i]);
    *reinterpret_cast<bf16x8*>(a.g + (size_t)(r0 + i) * a.ldg + c) = o;
  }
}

// ---------------------------------------------------------------------------------------------------- logits, streamed
// The logits of narrow layers (D <= 128, the width of this library's own layers): a tile has so few products that loading
// it, its softmax and its stores are what counts.  The tiles, 128 x 128, are dealt out to G workgroups in equal runs along the
// vocabulary; a wave keeps its 64 rows of h in registers for the run, and the words of the next tile arrive by LDS-DMA
// while this one is multiplied and exponentiated: one barrier per tile.  A lane keeps the running maximum and sum of its
// own columns of a row over the whole run; lanes, waves and workgroups are joined at its end.  Two workgroups per CU: one's
// vector instructions (max, fused multiply-add, exponential and sum per logit) run beside the other's products.  Stats of 3032
// x 128 x 32000: 42 us, g 61 us (as single tiles, each beginning with an empty pipeline, the stats took 109 us).  By the
// counters neither unit bounds it: of the stats' cycles the vector unit is given instructions in 0.51 and the matrix unit works
// in 0.30, of which 0.28 lie beside vector work, so in a third neither does anything; of g's 0.38 and 0.21.  The waves spend 0.31
// of their time waiting, for the tile that was requested one tile ago and at its barrier, and 0.30 and 0.39 ready but not
// issued, behind the other wave of the SIMD.
// A large vocabulary is cut into eight parts, one per XCD, so that the words that an XCD's workgroups read over and over stay
// in its L2 (all of 32000 x 128 from everywhere: 48 us, at the rate of the memory behind the L2s).
__host__ __device__ __forceinline__ int stream_parts(int qtiles) { return qtiles >= 64 ? 8 : 1; }
struct CeStream {
  int ptiles, qtiles, parts, per_part;   // tiles of the rows that count and of the vocabulary; workgroups per part
  int q0, qn, G;                         // this part's first tile of the vocabulary, how many, workgroups that have any
  uint32_t each, extra;                  // tiles per workgroup; the first `extra` have one more
  __device__ __forceinline__ CeStream(int rows, int V, int grid) {
    ptiles = (rows + 127) / 128;
    qtiles = (V + 127) / 128;
    parts = stream_parts(qtiles);
    per_part = parts == 8 ? grid >> 3 : grid;
  }
  __device__ __forceinline__ void part(int x) {
    q0 = parts == 8 ? (qtiles * x) >> 3 : 0;
    qn = (parts == 8 ? (qtiles * (x + 1)) >> 3 : qtiles) - q0;
    const uint32_t T = (uint32_t)ptiles * (uint32_t)qn;   // (the host keeps the tiles of a launch below 2^31)
    G = T < (uint32_t)per_part ? (int)T : per_part;
    each = G ? T / (uint32_t)G : 0;
    extra = T - each * (uint32_t)G;
  }
  __device__ __forceinline__ uint32_t begin(int b) const {
    return each * (uint32_t)b + ((uint32_t)b < extra ? (uint32_t)b : extra);
  }
  __device__ __forceinline__ int owner(uint32_t tile) const {
    const uint32_t longer = (each + 1) * extra;
    return (int)(tile < longer ? tile / (each + 1) : extra + (tile - longer) / each);
  }
  // where workgroup b of part x leaves its (max, sum) of the row tile pt, one of each half of the columns
  __device__ __forceinline__ size_t slot(int x, int b, int pt, int half) const {
    return (((size_t)x * (per_part + ptiles) + b + pt) * 2 + half) * 128;
  }
};

template <int MODE>
__global__ __launch_bounds__(256, 2) void ce_stream_kernel(const CeGemm a) {
  constexpr int MT = 4, NT = 4, KS = 4;   // 64 x 64 per wave, 128 of the contraction
  using OpQ = Operand<false, true, 128, 256, 64>;
  constexpr int STAGE = 2 * OpQ::BYTES;   // the two halves of the contraction
  constexpr bool STATS = MODE != LOGIT_GRAD;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[2 * STAGE];
  __shared__ float2 pair[MODE == LOGIT_LOSS ? 256 : 1];   // (max, sum) of a row's halves, its target's logit
  __shared__ float hit[MODE == LOGIT_LOSS ? 128 : 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rows = piece_rows(a);
  CeStream st(rows, a.Qn, gridDim.x);
  // workgroups go round the eight XCDs: one part each, or neighbours in the stream to one XCD
  const int xcd = blockIdx.x & 7, vocab_part = st.parts == 8 ? xcd : 0;
  const int b = st.parts == 8 ? (int)blockIdx.x >> 3 : xcd * ((int)gridDim.x >> 3) + ((int)blockIdx.x >> 3);
  st.part(vocab_part);
  if (b >= st.G) return;   // (uniform)
  const uint32_t t0 = st.begin(b);
  const int ntiles = (int)(st.begin(b + 1) - t0), qend = st.q0 + st.qn;
  int pt = (int)(t0 / (uint32_t)st.qn), qt = st.q0 + (int)(t0 - (uint32_t)pt * st.qn);
  const int pw0 = (wave >> 1) * 64, qw0 = (wave & 1) * 64;
  const int i16 = lane & 15, j4 = lane >> 4;
  const bool two = a.K > 64;
  lds_byte* const lds = (lds_byte*)smem;
  // the lane's source offsets in a tile of words, both halves of the contraction (past its end: past every bound)
  uint32_t off[2][OpQ::NI];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < OpQ::NI; ++i) {
      const int slot = i * 256 + tid, c = OpQ::piece(slot) + h * 8;
      off[h][i] = c * 8 < a.K ? (uint32_t)((slot / OpQ::ROW) * (int)a.ldq * 2 + c * 16) : OpQ::OUT;
    }
  auto words_of = [&](int q) {
    const int left = a.Qn - q * 128, n = left < 128 ? left : 128;
    return __builtin_amdgcn_make_buffer_rsrc((void*)(a.Q + (long)q * 128 * a.ldq), 0, ((n - 1) * (int)a.ldq + a.K) * 2, 0x00020000);
  };
  auto issue = [&](const __amdgpu_buffer_rsrc_t rsrc, lds_byte* wr, int h, int i) {   // instruction i of half h
    const lptr_t to = (lptr_t)(wr + h * OpQ::BYTES + i * 4096 + wave * 1024);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, to, 16, (int)off[h][i], 0, 0, 0);
  };
  {
    const __amdgpu_buffer_rsrc_t rsrc = words_of(qt);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < OpQ::NI; ++i) issue(rsrc, lds, h, i);
  }
  // The bias of the lane's columns, requested a tile ahead, 0 past the vocabulary and without a bias; nothing is done with
  // the values before that tile begins (a compare behind each load costs 16 memory latencies per tile: 71 us instead of 48).
  float raw[NT / 2][8];
  const __amdgpu_buffer_rsrc_t bias_rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)a.bias, 0, a.bias ? a.Qn * 4 : 0, 0x00020000);
  auto load_bias = [&](int q, int i) {   // instruction i of four
    const int at = (q * 128 + qw0 + 8 * j4) * 4 + (i >> 1) * 128 + (i & 1) * 16;
    const f32x4 v = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(bias_rsrc, at, 0, 0));
#pragma unroll
    for (int e = 0; e < 4; ++e) raw[i >> 1][(i & 1) * 4 + e] = v[e];
  };
  float m2[MT], sum[MT], lse2[MT], wt[MT];   // running maximum and sum; lse in units of log 2 and weight (gradient)
  int target[MT];
  bool far = false;   // the rows' maxima are too large for one multiply-add
  bf16x8 pf[MT][KS];
  auto load_rows = [&](int p) {   // (no branch around a load: each would be waited for before the next)
    const int left = rows - p * 128, n = left < 128 ? left : 128;
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)(a.P + (long)p * 128 * a.ldp), 0,
                                                                          ((n - 1) * (int)a.ldp + a.K) * 2, 0x00020000);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int r = pw0 + mt * 16 + i16, m = p * 128 + (r < n ? r : n - 1);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int k = ks * 32 + 8 * j4;
        const int at = k < a.K ? (r * (int)a.ldp + k) * 2 : (int)OpQ::OUT;
        pf[mt][ks] = __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(rsrc, at, 0, 0));
      }
      target[mt] = a.word ? a.word[m] : (int)(a.target[m] >= 0 && a.target[m] < a.Qn ? a.target[m] : -1);
      if (MODE == LOGIT_GRAD) {
        const float2 l = a.lse[m];
        lse2[mt] = l.x;
        sum[mt] = l.y;
        wt[mt] = a.weight[m];
      }
    }
    far = false;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const bool there = pw0 + mt * 16 + i16 < n;
      m2[mt] = -INFINITY;
      if (STATS) sum[mt] = 0.f;
      target[mt] = there && target[mt] >= 0 ? target[mt] : -1 << 30;
      if (MODE == LOGIT_GRAD) {   // a row that is not there, or whose every logit is masked: no gradient
        const bool live = there && sum[mt] != -INFINITY;
        far |= live && fabsf(lse2[mt]) > FAR;
        lse2[mt] = live ? __builtin_fmaf(lse2[mt], LOG2E, sum[mt]) : INFINITY;
        wt[mt] = live ? wt[mt] : 0.f;
      }
    }
    // A use of all of it, here: the compiler waits for a loaded value where it is first used, and in the loop that would be
    // a wait for everything requested since, once per tile.
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      asm volatile("" : "+v"(target[mt]));
      if (MODE == LOGIT_GRAD) asm volatile("" : "+v"(lse2[mt]), "+v"(wt[mt]));
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(pf[mt][ks]));
    }
  };
  auto bias_arrived = [&]() {   // (the same)
#pragma unroll
    for (int tp = 0; tp < NT / 2; ++tp)
#pragma unroll
      for (int e = 0; e < 8; ++e) asm volatile("" : "+v"(raw[tp][e]));
  };
  load_rows(pt);
#pragma unroll
  for (int i = 0; i < 4; ++i) load_bias(qt, i);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  bias_arrived();

  for (int t = 0; t < ntiles; ++t) {
    const int q0 = qt * 128;
    const bool new_rows = qt + 1 == qend, more = t + 1 < ntiles;
    const int pt1 = new_rows ? pt + 1 : pt, qt1 = new_rows ? st.q0 : qt + 1;
    // The products start from the bias: -infinity past the vocabulary, which leaves those columns out of everything.
    f32x4 start[NT];
    if (q0 + 128 > a.Qn)
#pragma unroll
      for (int tp = 0; tp < NT / 2; ++tp)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (q0 + qw0 + tp * 32 + 8 * j4 + e >= a.Qn) raw[tp][e] = -INFINITY;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) start[nt][e] = raw[nt >> 1][(nt & 1) * 4 + e];
    // (this wave's share of the tile has landed, see below: behind the barrier everybody's has, and nobody reads the other stage)
    asm volatile("s_barrier" ::: "memory");
    f32x4 acc[MT][NT];
    [&](lds_byte* __restrict__ wr, const lds_byte* __restrict__ rd) {
      // The next tile's requests go between the products, since in one go they would hold those up (four waves' twelve
      // instructions at 18 cycles each of the address unit).  A run's last tile requests itself again and nobody looks.
      const int q1 = more ? qt1 : qt;
      const __amdgpu_buffer_rsrc_t rsrc = words_of(q1);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        bf16x8 qf[NT];
        if (ks < 2 || two)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            qf[nt] = OpQ::frag(rd + (ks >> 1) * OpQ::BYTES, qw0 + (nt >> 1) * 32, nt & 1, ks & 1, lane);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          if (ks < 2 || two)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              acc[mt][nt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(qf[nt], pf[mt][ks], ks ? acc[mt][nt] : start[nt], 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
          const int k = ks * MT + mt;   // 16 places
          if (k < 8) issue(rsrc, wr, k >> 2, k & 3);
          else if (k < 12) load_bias(q1, k - 8);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }(lds + (~t & 1) * STAGE, lds + (t & 1) * STAGE);
    // the lane's column of the target's logit is 0..7 or 32..39 of the wave's; most tiles hold no row's target
    const int base = q0 + qw0 + 8 * j4;
    bool any = false;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) any |= ((target[mt] - base) & ~39) == 0;
    const bool targets = __ballot(any) != 0;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      if constexpr (STATS) {
        float v = acc[mt][0][0];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) v = fmaxf(v, acc[mt][nt][e]);
        const float top = fmaxf(m2[mt], v), at = top == -INFINITY ? 0.f : top;   // nothing but masked words so far
        float x = sum[mt] * __builtin_amdgcn_exp2f((m2[mt] - at) * LOG2E);
        if (__ballot(fabsf(at) > FAR)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) x += __builtin_amdgcn_exp2f((acc[mt][nt][e] - at) * LOG2E);
        } else {
          const float at2 = at * LOG2E;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) x += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[mt][nt][e], LOG2E, -at2));
        }
        m2[mt] = top;
        sum[mt] = x;
      } else {
        float l2 = lse2[mt];
        if (__ballot(far)) {   // (the lse again, its two parts)
          const int m = pt * 128 + pw0 + mt * 16 + i16;
          const float2 l = a.lse[m < rows ? m : rows - 1];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[mt][nt][e] -= l.x == -INFINITY ? 0.f : l.x;
          l2 = l2 == INFINITY ? l2 : l.y;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            acc[mt][nt][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[mt][nt][e], LOG2E, -l2)) * wt[mt];
        if (targets)
#pragma unroll
          for (int tp = 0; tp < NT / 2; ++tp)
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[mt][2 * tp + (e >> 2)][e & 3] -= target[mt] - base == tp * 32 + e ? wt[mt] : 0.f;
      }
    }
    // The next tile's words have landed (they had this tile's products and exponentials to do so, which is why those are made
    // to be done here); waited for here and not at the barrier, which would wait for the following stores as well.  So are this
    // tile's LDS reads, behind which the next barrier lets its stage be written.
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      if constexpr (STATS) asm volatile("" : "+v"(sum[mt]), "+v"(m2[mt]));
      else
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) asm volatile("" : "+v"(acc[mt][nt]));
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    bias_arrived();
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int m = pt * 128 + pw0 + mt * 16 + i16;
      if constexpr (STATS) {
        if (targets) {
          float x = 0.f;
#pragma unroll
          for (int tp = 0; tp < NT / 2; ++tp)
#pragma unroll
            for (int e = 0; e < 8; ++e) x = target[mt] - base == tp * 32 + e ? acc[mt][2 * tp + (e >> 2)][e & 3] : x;
          if (((target[mt] - base) & ~39) == 0) {
            if (MODE == LOGIT_LOSS) hit[pw0 + mt * 16 + i16] = x;
            else a.tlogit[m] = x;
          }
        }
      } else if (m < rows) {
#pragma unroll
        for (int tp = 0; tp < NT / 2; ++tp) {
          bf16x8 o;
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = (bf16)acc[mt][2 * tp + (e >> 2)][e & 3];
          *reinterpret_cast<bf16x8*>(a.g + (size_t)m * a.ldg + q0 + qw0 + tp * 32 + 8 * j4) = o;
        }
      }
    }
    if (new_rows || !more) {
      if constexpr (STATS) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const float top = xor32_max(xor16_max(m2[mt])), at = top == -INFINITY ? 0.f : top;
          const float x = xor32_sum(xor16_sum(sum[mt] * __builtin_amdgcn_exp2f((m2[mt] - at) * LOG2E)));
          if (j4 == 0) {
            float2* to = MODE == LOGIT_LOSS ? pair + (wave & 1) * 128 : a.part + st.slot(vocab_part, b, pt, wave & 1);
            to[pw0 + mt * 16 + i16] = make_float2(top, x);
          }
        }
        if (MODE == LOGIT_LOSS) {   // (the next tile's barrier keeps its pairs from overtaking these)
          __syncthreads();
          const int m = pt * 128 + tid;
          if (tid < 128 && m < rows) {
            const float2 p = pair[tid], q = pair[128 + tid];
            const float top = fmaxf(p.x, q.x), at = top == -INFINITY ? 0.f : top;
            const float x = p.y * __builtin_amdgcn_exp2f((p.x - at) * LOG2E) + q.y * __builtin_amdgcn_exp2f((q.x - at) * LOG2E);
            const float s = logf(x), l = at + s;
            const int64_t t = a.target[m];
            const bool none = t == a.ignore, word = t >= 0 && t < a.Qn;
            a.loss_out[m] = none ? 0.f : !word ? __builtin_nanf("") : l == -INFINITY ? INFINITY : s + (at - hit[tid]);
            if (a.lse_out) a.lse_out[m] = none ? 0.f : !word ? __builtin_nanf("") : l;
          }
        }
      }
      if (more) load_rows(pt1);
    }
    pt = pt1;
    qt = qt1;
  }
}

// ---------------------------------------------------------------------------------------------------- rows
// The rows that count, numbered through in their order (one workgroup: 16 waves look at 1024 targets at a time), and the
// losses of those that do not: 0 where the target is ignore_index, NaN where it is no word (and no gradient).  The largest weight.
__global__ __launch_bounds__(1024) void ce_index_kernel(const int64_t* target, int64_t ignore, int N, int V, int* index,
                                                        int* words, int* count, float* loss, float* lse, const float* dloss,
                                                        float scale, float* unit) {
  __shared__ int waves[16];
  __shared__ float top[16];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int done = 0;
  float largest = 0.f;   // (NaN does not count)
  for (int base = 0; base < N; base += 1024) {
    const int n = base + (int)threadIdx.x;
    int64_t t = ignore;
    float wt = 1.f;
    if (n < N) {
      t = target[n];
      if (dloss) wt = dloss[n];
    }
    const bool word = t >= 0 && t < V, keep = n < N && t != ignore && word;
    if (n < N && !keep) {
      const float x = t == ignore ? 0.f : __builtin_nanf("");
      loss[n] = x;
      if (lse) lse[n] = x;
    }
    const unsigned long long b = __ballot(keep);
    __syncthreads();
    if (lane == 0) waves[w] = __popcll(b);
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int c = waves[i];
      before += i < w ? c : 0;
      all += c;
    }
    if (keep) {
      largest = fmaxf(largest, fabsf(scale * wt));
      const int at = done + before + __popcll(b & ((1ull << lane) - 1));
      index[at] = n;
      words[at] = (int)t;
    }
    done += all;
  }
  largest = wave_max(largest);
  if (lane == 0) top[w] = largest;
  __syncthreads();
  if (threadIdx.x != 0) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) largest = fmaxf(largest, top[i]);
  *count = done;
  *unit = largest > 0.f && largest < INFINITY ? largest : 1.f;   // (a weight of infinity stays with its row)
}

// A piece's rows, one after another (16 bytes per lane), and their weights; behind its `gather` workgroups those that clear dh
// of the rows that do not count, 16 rows each.  (The loss alone has neither weights nor dh, here and below.)
__global__ __launch_bounds__(256) void ce_gather_kernel(const bf16* h, long ldh, int D8, const int* index, const int* count,
                                                        int row0, int rows_max, const float* dloss, float scale, bf16* out,
                                                        float* weight, const float* unit, unsigned gather,
                                                        const int64_t* target, int64_t ignore, int N, int V, bf16* dh,
                                                        long lddh) {
  if (blockIdx.x >= gather) {
    const long n = (long)(blockIdx.x - gather) * 16 + (threadIdx.x >> 4);
    if (n >= N) return;
    const int64_t t = target[n];
    if (t != ignore && t >= 0 && t < V) return;
    for (int c = threadIdx.x & 15; c < D8; c += 16) reinterpret_cast<uint4*>(dh + n * lddh)[c] = make_uint4(0, 0, 0, 0);
    return;
  }
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  const int r = (int)(i / D8), c = (int)(i - (long)r * D8);
  int rows = *count - row0;
  rows = rows < rows_max ? rows : rows_max;
  if (r >= rows) return;
  const int n = index[row0 + r];
  if (c == 0 && weight) weight[r] = scale * (dloss ? dloss[n] : 1.f) / *unit;
  reinterpret_cast<uint4*>(out)[(long)r * D8 + c] = reinterpret_cast<const uint4*>(h + (long)n * ldh)[c];
}

// Both of these in one launch, for few rows in one piece: a workgroup has 16 rows, 16 lanes each, and looks at all the targets
// and weights itself, for the number of rows that count before its own and the largest weight.  That grows with the square of
// the rows, so up to MERGE_ROWS.  All of the gradient, in one launch / in two: 64 x 128 x 43 24 / 27 us, 4032 x 128 x 43 32 /
// 35, 8192 x 1024 x 43 63 / 71, 16384 x 128 x 43 61 / 64, 32768 x 128 x 43 98 / 96, 65536 x 128 x 43 211 / 150.
__global__ __launch_bounds__(256) void ce_index_gather_kernel(const bf16* h, long ldh, int D8, const int64_t* target,
                                                              int64_t ignore, int N, int V, const float* dloss, float scale,
                                                              int* index, int* words, int* count, float* unit, float* weight,
                                                              bf16* out, float* loss, float* lse, bf16* dh, long lddh) {
  __shared__ int before_of[4], all_of[4];
  __shared__ float top_of[4];
  const int tid = threadIdx.x, w = tid >> 6, first = blockIdx.x * 16;
  int before = 0, all = 0;
  float largest = 0.f;   // (NaN does not count)
#pragma unroll 4
  for (int n = tid; n < N; n += 256) {
    const int64_t t = target[n];
    const float wt = fabsf(scale * (dloss ? dloss[n] : 1.f));
    const bool keep = t != ignore && t >= 0 && t < V;
    all += keep;
    before += keep && n < first;
    largest = fmaxf(largest, keep ? wt : 0.f);
  }
  const int lane = tid & 63;
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    all += __shfl_xor(all, d);
    before += __shfl_xor(before, d);
  }
  largest = wave_max(largest);
  if (lane == 0) { all_of[w] = all; before_of[w] = before; top_of[w] = largest; }
  __syncthreads();
  largest = fmaxf(fmaxf(top_of[0], top_of[1]), fmaxf(top_of[2], top_of[3]));
  const float most = largest > 0.f && largest < INFINITY ? largest : 1.f;   // (a weight of infinity stays with its row)
  if (blockIdx.x == 0 && tid == 0) {
    *count = all_of[0] + all_of[1] + all_of[2] + all_of[3];
    *unit = most;
  }
  // lane i of each wave knows of row i: which of the 16 count
  int64_t mine = ignore;
  if (lane < 16 && first + lane < N) mine = target[first + lane];
  const unsigned long long rows = __ballot(lane < 16 && first + lane < N && mine != ignore && mine >= 0 && mine < V);
  const int r = tid >> 4, n = first + r;
  if (n >= N) return;
  const int64_t t = target[n];
  if ((rows >> r) & 1) {
    const int at = before_of[0] + before_of[1] + before_of[2] + before_of[3] + __popcll(rows & ((1ull << r) - 1));
    if ((tid & 15) == 0) {
      index[at] = n;
      words[at] = (int)t;
      if (weight) weight[at] = scale * (dloss ? dloss[n] : 1.f) / most;
    }
    for (int c = tid & 15; c < D8; c += 16)
      reinterpret_cast<uint4*>(out)[(long)at * D8 + c] = reinterpret_cast<const uint4*>(h + (long)n * ldh)[c];
  } else {
    if ((tid & 15) == 0) {
      const float x = t == ignore ? 0.f : __builtin_nanf("");
      loss[n] = x;
      if (lse) lse[n] = x;
    }
    if (dh)
      for (int c = tid & 15; c < D8; c += 16) reinterpret_cast<uint4*>(dh + (long)n * lddh)[c] = make_uint4(0, 0, 0, 0);
  }
}

// A row's pairs (maximum, sum) -> lse and loss: 16 rows per workgroup, 16 lanes each.  The pairs are those
// of every 64 words, [.][ld], or (grid != 0) those that the workgroups of ce_stream_kernel left.
__global__ __launch_bounds__(256) void ce_rows_kernel(const float2* part, int tiles, int ld, int grid, const int* count, int row0,
                                                      int rows_max, const int* index, const int64_t* target, int64_t ignore,
                                                      int V, const float* tlogit, float2* lse_c, float* loss, float* lse) {
  __shared__ float rm[16][16], rs[16][16];
  int rows = rows_max;
  if (count) {
    rows = *count - row0;
    rows = rows < rows_max ? rows : rows_max;
  }
  const int i = threadIdx.x & 15, j = threadIdx.x >> 4, r = blockIdx.x * 16 + i;
  if ((int)blockIdx.x * 16 >= rows) return;
  float m = -INFINITY, s = 0.f;
  auto join = [&](const float2 p) {
    const float top = fmaxf(m, p.x), at = top == -INFINITY ? 0.f : top;
    s = s * __builtin_amdgcn_exp2f((m - at) * LOG2E) + p.y * __builtin_amdgcn_exp2f((p.x - at) * LOG2E);
    m = top;
  };
  if (r < rows && !grid) {
    int q = j;
    for (; q + 112 < tiles; q += 128) {   // eight at a time: their loads are in flight together, and one new maximum
      float2 p[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) p[k] = part[(size_t)(q + 16 * k) * ld + r];
      float top = m;
#pragma unroll
      for (int k = 0; k < 8; ++k) top = fmaxf(top, p[k].x);
      const float at = top == -INFINITY ? 0.f : top;
      s *= __builtin_amdgcn_exp2f((m - at) * LOG2E);
#pragma unroll
      for (int k = 0; k < 8; ++k) s += p[k].y * __builtin_amdgcn_exp2f((p[k].x - at) * LOG2E);
      m = top;
    }
    for (; q < tiles; q += 16) join(part[(size_t)q * ld + r]);
  }
  if (r < rows && grid) {   // lane j: part j / 2 (or j of 16 lanes the only one), half j & 1 of the columns
    CeStream st(rows, V, grid);
    const int pt = (int)blockIdx.x / 8, x = st.parts == 8 ? j >> 1 : 0;
    st.part(x);
    const int b0 = st.owner((uint32_t)pt * st.qn), b1 = st.owner((uint32_t)(pt + 1) * st.qn - 1);
    for (int b = b0 + (st.parts == 8 ? 0 : j >> 1); b <= b1; b += st.parts == 8 ? 1 : 8)
      join(part[st.slot(x, b, pt, j & 1) + (r & 127)]);
  }
  rm[j][i] = m;
  rs[j][i] = s;
  __syncthreads();
  if (j != 0 || r >= rows) return;
  float top = m;
#pragma unroll
  for (int k = 1; k < 16; ++k) top = fmaxf(top, rm[k][i]);
  const float at = top == -INFINITY ? 0.f : top;
  float all = 0.f;
#pragma unroll
  for (int k = 0; k < 16; ++k) all += rs[k][i] * __builtin_amdgcn_exp2f((rm[k][i] - at) * LOG2E);
  const float ls = logf(all);
  float l = at + ls;   // all == 0: -inf, every logit of the row is masked
  if (lse_c) lse_c[r] = make_float2(top, log2f(all));
  const int n = index ? index[row0 + r] : r;
  float x;
  const int64_t t = target[n];
  if (!index && (t == ignore || t < 0 || t >= V)) x = l = t == ignore ? 0.f : __builtin_nanf("");
  else x = l == -INFINITY ? INFINITY : ls + (at - tlogit[r]);   // (at and the logit may be far larger than the loss)
  loss[n] = x;
  if (lse) lse[n] = l;
}

// The results of a product from the slabs of its split contraction: 4 columns per lane, behind them the words of dbias
template <int MODE> __device__ __forceinline__ void join_slabs(const CeGemm& a, long i) {
  const int D4 = a.Qn / 4, rows = MODE == DH ? piece_rows(a) : a.Pn;
  const long r = i / D4;
  const size_t c = (size_t)(i - r * D4) * 4, stride = (size_t)a.Pn * a.ldslab;
  const float unit = *a.unit;
  if (r < rows) {
    const float* p = a.slab + (size_t)r * a.ldslab + c;
    f32x4 s = *reinterpret_cast<const f32x4*>(p);
    for (int k = 1; k < a.ksplit; ++k) s += *reinterpret_cast<const f32x4*>(p + k * stride);
    s *= unit;
    if (MODE == DW && a.acc_in) s += *reinterpret_cast<const f32x4*>(a.acc_in + (size_t)r * a.Qn + c);
    const size_t at = (size_t)(MODE == DH ? a.index[r] : (int)r) * a.ldo + c;
    if (MODE == DW && a.out_f32) {
      *reinterpret_cast<f32x4*>((float*)a.out + at) = s;
    } else {
      bf16x4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = (bf16)s[e];
      *reinterpret_cast<bf16x4*>((bf16*)a.out + at) = o;
    }
  }
  if (MODE == DW && a.dbias) {
    const long v = i - (long)a.Pn * D4;
    if (v < 0 || v >= a.Pn) return;
    float s = a.slab_bias[v];
    for (int k = 1; k < a.ksplit; ++k) s += a.slab_bias[(size_t)k * a.Pn + v];
    s *= unit;
    if (a.dbias_in) s += a.dbias_in[v];
    if (a.dbias_f32) ((float*)a.dbias)[v] = s;
    else ((bf16*)a.dbias)[v] = (bf16)s;
  }
}

__global__ __launch_bounds__(256) void ce_slabs_kernel(const CeGemm dh, const CeGemm dw, unsigned n) {   // n workgroups for dh
  if (blockIdx.x < n) join_slabs<DH>(dh, (long)blockIdx.x * 256 + threadIdx.x);
  else join_slabs<DW>(dw, (long)(blockIdx.x - n) * 256 + threadIdx.x);
}

// ---------------------------------------------------------------------------------------------------- host
struct CePlan {
  long rows;          // per piece, a multiple of 256
  int pieces, split_dh, split_dw;
  bool stream, whole; // logits: ce_stream_kernel; with the loss in it
  bool number;        // the rows that count are numbered through and gathered
  bool big, wide;     // or tiles of 256 x 256, of 128 x 160 (loss); otherwise 128 x 128
  bool few;           // of these at most one per CU: four stages of LDS (loss of 200 x 4096 x 1000 uncut: 41 us, 46 with two)
  int split_logits;   // or in parts of the contraction, joined by ce_join_kernel
  bool big_dh, big_dw;
  int parts, pairs;   // logits: parts of the vocabulary of the stream; (maximum, sum) per row otherwise: one per 64 words, or 160
  long Vp;
  size_t index, words, tlogit, lse, weight, part, hc, g, slab_logits, slab_dh, slab_dw, slab_bias, dwacc, dbacc, total;
};

constexpr int STREAM_GRID = 512, TILE_GRID = 256;   // two workgroups per CU, one
constexpr double NUMBER_PART = 1.0 / 16;
constexpr int JOIN_VOCAB = 8192, MERGE_ROWS = 16384;
constexpr size_t PIECE_BYTES = (size_t)4 << 30;   // g of a piece, unless the caller says how many rows
constexpr size_t PIECE_MAX = (size_t)64 << 30, HC_MAX = (size_t)16 << 30;   // g and the rows of h, in any case
constexpr size_t PAIR_BYTES = (size_t)1 << 30;    // pairs of a piece, where only the loss is asked for
constexpr size_t STREAM_PAIRS = (size_t)STREAM_GRID * 2 * 128 * 8;   // of the stream, where it has no rows

bool dw_f32(const mmst_linear_ce_args* a) { return a->grad_f32 && a->grad_f32 != 2; }

bool sizes_ok(const mmst_linear_ce_args* a) {
  return a && a->N >= 0 && a->N <= MMST_LINEAR_CE_MAX_ROWS && a->V >= 1 && a->V <= MMST_LINEAR_CE_MAX_VOCAB && a->D >= 8 &&
         a->D % 8 == 0 && a->D <= MMST_LINEAR_CE_MAX_DIM && a->rows_per_piece >= 0 &&
         (((long)a->N + 127) / 128) * (((long)a->V + 127) / 128) < 0x7FFFFFFFL;   // tiles of one launch
}

bool args_ok(const mmst_linear_ce_args* a, bool grad) {
  if (!sizes_ok(a)) return false;
  auto rows_ok = [&](const void* p, long ld, long n) {
    return p && (uintptr_t)p % 16 == 0 && ld % 8 == 0 && (n <= 1 || ld >= a->D) && ld <= MMST_LINEAR_CE_MAX_LD;
  };
  if (!rows_ok(a->w, a->ldw, a->V)) return false;
  if (a->N > 0 && (!rows_ok(a->h, a->ldh, a->N) || !a->target || !a->loss)) return false;
  auto aligned = [](const void* p, size_t n) { return (uintptr_t)p % n == 0; };   // (NULL is)
  if (!aligned(a->target, 8) || !aligned(a->bias, 4) || !aligned(a->loss, 4) || !aligned(a->lse, 4)) return false;
  if (!grad) return true;
  if (!aligned(a->dloss, 4) || !aligned(a->dbias, a->grad_f32 ? 4 : 2)) return false;
  return (a->N == 0 || rows_ok(a->dh, a->lddh, a->N)) && a->dw && (uintptr_t)a->dw % 16 == 0;
}

size_t align(size_t x) { return (x + 255) & ~(size_t)255; }

long tiles(long n, long m, int b) { return ((n + b - 1) / b) * ((m + b - 1) / b); }

// 256 x 256 tiles, one workgroup per CU, or 128 x 128, two: whichever is done first.  A round of the small ones (512 tiles,
// half as much work) takes 14 / 26 of a round of the large ones, whose steps feed the matrix units better, and three fifths of
// that where no CU has more than one; what a last, partly filled round wastes decides.  Measured, large / small: the loss at
// 2048 x 1024 x 16384 (rows, width, words; 2 rounds against 4) 70 / 78 us, at 333 x 1024 x 50001 (2 against 2 and 149 tiles) 68 /
// 55 us; all of the gradient with dw by either at 8192 x 1024 x 32000 (2 against 4) 1696 / 1820 us, at 4096 x 256 x 8192 (1
// against 128 tiles) 192 / 158 us.
long fifths(long t) {   // of a round of two workgroups per CU
  const long rest = t % (2 * TILE_GRID);
  return t / (2 * TILE_GRID) * 5 + (rest == 0 ? 0 : rest <= TILE_GRID ? 3 : 5);
}
long cost_large(long n, long m) { return 26 * 5 * ((tiles(n, m, 256) + TILE_GRID - 1) / TILE_GRID); }
long cost_small(long n, long m) { return 14 * fifths(tiles(n, m, 128)); }
bool large_tiles(long n, long m) { return cost_large(n, m) <= cost_small(n, m); }

// For the loss alone also 128 rows x 160 words, whose rounds take 17 / 26: measured, 160 words / what is taken without them: 333 x
// 1024 x 50001 (2 rounds against 3 of 128) 50 / 54 us, 333 x 4096 x 50001 190 / 222, 128 x 2048 x 80000 83 / 104, 200 x 2048 x
// 40000 49 / 62, 512 x 1024 x 20000 31 / 37, 1000 x 1024 x 10000 29 / 36, 512 x 2048 x 50001 111 / 124, 333 x 256 x 80000 32 / 38,
// 1000 x 1024 x 40000 95 / 98, 2000 x 2048 x 20000 168 / 172, 3000 x 512 x 10000 44.6 / 45.0, 64 x 1024 x 100000 48 / 48, 512 x 512 x
// 10000 15.9 / 15.6.
bool wide_tiles(long n, long m) {
  const long wide = 17 * fifths((n + 127) / 128 * ((m + 159) / 160));
  return wide < cost_large(n, m) && wide < cost_small(n, m);
}

// Parts of a contraction (of dh: the vocabulary, of dw: the rows), each of at least eight steps: as many as are done first,
// counted in steps of the workgroups that run at once (`slots`: one per CU with large tiles; with small ones two, or one of each
// product where both are in one launch) and what writing and reading the fp32 slabs takes, 1 / 10 of a step per large tile and
// part, 1 / 20 per small one.  All of the gradient of 4032 x 128 x 43: 72 us with dw uncut, 45 in 7 parts (in launches of their
// own); of 3032 x 128 x 32000 in one launch: 189 us for 4 parts of dh, 167 for 8, 197 for 16; of 10878 x 568 x 41518 2970 us for
// one (129 tiles), 2610 for 3; of 1840 x 680 x 773 67 us for as many as fill the slots once, 46 for the best.
struct Parts { int n; double steps; };
Parts parts(long t, bool big, long slots, long contraction) {
  const long steps = (contraction + 63) / 64;
  const double join = big ? 1.0 / 10 : 1.0 / 20;
  Parts best = {1, (double)((t + slots - 1) / slots * steps)};
  for (long s = 2; s <= 32 && s <= steps / 8; ++s) {
    const double cost = (double)((t * s + slots - 1) / slots) * (double)steps / (double)s + (double)(t * s) * join;
    if (cost < best.steps) best = {(int)s, cost};
  }
  return best;
}

// Parts of the logits' contraction (`steps` of it) where t tiles leave most CUs idle: at least eight steps each, and more than 16
// steps (of half a microsecond) fewer in a row, which pays for the join.  Loss, uncut / in parts: 64 x 4096 x 43 (8 parts) 41 / 17
// us, 200 x 4096 x 1000 (8) 41 / 20, 16 x 2048 x 8000 (4) 27 / 18, 500 x 2000 x 3000 (2, 16 steps fewer) 26 / 28; with four steps
// each, 16 parts, 200 x 4096 x 1000 takes 23.
int logit_parts(long t, long steps) {
  if (t == 0) return 1;
  long s = TILE_GRID / t;
  if (s > steps / 8) s = steps / 8;
  return s >= 2 && steps - steps / s > 16 ? (int)s : 1;
}

// Narrow layers: the stream where a workgroup gets more than two tiles of it, for which it computes the logits twice and
// reads no exponentials back.  Measured, stream / tiles, loss and gradient: 3000 x 128 x 8000 (1512 tiles) 19 / 23 and 93 / 97
// us, 3000 x 128 x 32000 42 / 65 and 193 / 239, 2000 x 128 x 8000 (1008) 19 / 16 and 80 / 79, 512 x 128 x 4000 (128) 15 / 14
// and 55 / 47.
bool streams(long n, const mmst_linear_ce_args* a) { return a->D <= 128 && tiles(n, a->V, 128) > 2 * STREAM_GRID; }

// The loss alone: rows that do not count are numbered out where that, estimated in nanoseconds and as if none could be left
// out, takes at most NUMBER_PART of the products.  Measured, every row in the products / numbered through, of 0 and of half
// the rows ignored: 4032 x 128 x 32000 47, 47 / 54, 37 us; 1000 x 1024 x 50001 110, 107 / 118, 64; 65536 x 128 x 32000 577, 574 /
// 639, 356; 1000000 x 256 x 1000 944, 932 / 1993, 1526 (by the estimate not numbered); 2000 x 1024 x 50001 221, 206 / 226, 116;
// 4032 x 1024 x 50001 377, 378 / 366, 206; 8192 x 2048 x 65536 1729, 1720 / 1735, 865; 4096 x 4096 x 32000 831, 827 / 843, 432.
bool numbers(long n, long d, long v) {
  const double products = (double)n * (double)v * (1e-4 + (double)d * 2 / 1.3e6), numbering = 6000 + n * (1 + (double)d / 5000);
  return numbering <= products * NUMBER_PART;
}

CePlan plan(const mmst_linear_ce_args* a, bool grad) {
  CePlan p = {};
  p.Vp = ((long)a->V + VT - 1) / VT * VT;
  const long all = ((long)a->N + 255) / 256 * 256;
  auto limit = [&](size_t bytes, size_t row) {   // rows of a piece, so that `row` bytes of each are no more than `bytes`
    const long fit = (long)(bytes / row) / 256 * 256;
    p.rows = p.rows < fit ? p.rows : fit < 256 ? 256 : fit;
  };
  p.rows = all ? all : 256;
  p.parts = stream_parts((a->V + 127) / 128);
  p.whole = !grad && a->D <= 128 && a->V <= 128;
  p.stream = p.whole || (!grad && streams(a->N, a));
  p.number = grad || (!p.whole && numbers(a->N, a->D, a->V));
  if (grad) {
    if (a->rows_per_piece) limit(((size_t)a->rows_per_piece + 255) / 256 * 256, 1);
    else limit(PIECE_BYTES, p.Vp * 2);
    limit(PIECE_MAX, p.Vp * 2);
    limit(HC_MAX, (size_t)a->D * 2);
  } else if (p.stream && !p.whole) {   // what CeStream::slot counts: two pairs per row and part of the vocabulary
    limit(PAIR_BYTES - STREAM_PAIRS, (size_t)p.parts * 16);
  } else if (!p.whole) {
    limit(PAIR_BYTES, (size_t)((a->V + 255) / 256 * 4) * 8);
  }
  if (!grad && p.number) limit(PAIR_BYTES, (size_t)a->D * 2);
  p.pieces = all ? (int)((all + p.rows - 1) / p.rows) : 1;
  const long rows = a->N < p.rows ? a->N : p.rows;
  if (grad) p.stream = streams(rows, a);
  p.big = large_tiles(rows, a->V);
  p.wide = !grad && wide_tiles(rows, a->V);
  p.few = tiles(rows, a->V, 128) <= TILE_GRID;
  p.split_logits = p.stream ? 1 : logit_parts(tiles(rows, a->V, 128), (a->D + 63) / 64);
  if (grad) {
    p.big_dw = large_tiles(a->V, a->D);
    // A step of small tiles takes 7 / 13 of one of large ones; large ones for dh also where they take 5 % more by that count.
    // Measured, large / small: 2048 x 512 x 32000 (16 large tiles) 311 / 300 us, 1400 x 1024 x 50001 (24) 533 / 548, 8192 x 1024 x
    // 32000 (128) 1696 / 1791.
    const long slots = p.big_dw ? 2 * TILE_GRID : TILE_GRID;   // of small tiles, beside dw or alone
    const Parts large = parts(tiles(rows, a->D, 256), true, TILE_GRID, a->V);
    const Parts small = parts(tiles(rows, a->D, 128), false, 2 * TILE_GRID, a->V);
    p.big_dh = large.steps * 13 <= small.steps * 7 * 1.05;
    p.split_dh = p.big_dh ? large.n : parts(tiles(rows, a->D, 128), false, slots, a->V).n;
    p.split_dw = p.big_dw ? parts(tiles(a->V, a->D, 256), true, TILE_GRID, rows).n
                          : parts(tiles(a->V, a->D, 128), false, p.big_dh ? 2 * TILE_GRID : TILE_GRID, rows).n;
  }
  size_t at = 256;   // count, unit
  auto take = [&](size_t n) { const size_t o = at; at += align(n); return o; };
  if (p.split_logits > 1) p.slab_logits = take((size_t)p.split_logits * p.rows * ((a->V + 7) & ~7) * 4);
  p.pairs = p.split_logits > 1 ? (a->V + 63) / 64 : p.wide ? (a->V + 159) / 160 : p.big ? (a->V + 255) / 256 * 4
                                                                                       : (a->V + 127) / 128 * 2;
  if (!p.whole) {   // (which keeps both in LDS)
    p.tlogit = take(p.rows * 4);
    p.part = take(p.stream ? STREAM_PAIRS + (size_t)p.parts * 16 * p.rows : (size_t)p.pairs * p.rows * 8);
  }
  if (p.number) {
    p.index = take((size_t)(all + 256) * 4);
    p.words = take((size_t)(all + 256) * 4);
    p.hc = take((size_t)p.rows * a->D * 2);
  }
  if (grad) {
    p.lse = take(p.rows * 8);
    p.weight = take(p.rows * 4);
    p.g = take((size_t)p.rows * p.Vp * 2);
    const size_t dh = p.split_dh > 1 ? (size_t)p.split_dh * p.rows : 0, dw = p.split_dw > 1 ? (size_t)p.split_dw * a->V : 0;
    if (dh) p.slab_dh = take(dh * a->D * 4);
    if (dw) p.slab_dw = take(dw * a->D * 4);
    if (dw) p.slab_bias = take(dw * 4);
    if (p.pieces > 1 && !dw_f32(a)) p.dwacc = take((size_t)a->V * a->D * 4);
    if (p.pieces > 1 && !a->grad_f32 && a->dbias) p.dbacc = take((size_t)a->V * 4);
  }
  p.total = at;
  return p;
}

template <int MODE> void launch_product(const CeGemm& g, bool big, unsigned grid, hipStream_t st) {
  if (big) hipLaunchKernelGGL((ce_product_kernel<MODE, 256, 256, 2, 4>), dim3(grid), dim3(512), 0, st, g);
  else hipLaunchKernelGGL((ce_product_kernel<MODE, 128, 128, 2, 2>), dim3(grid), dim3(256), 0, st, g);
}
int launch_products(CeGemm& dh, CeGemm& dw, const CePlan& p, hipStream_t st) {
  auto grid = [](CeGemm& g, bool big) {
    const int b = big ? 256 : 128;
    g.ptiles = (g.Pn + b - 1) / b;
    g.qtiles = (g.Qn + b - 1) / b;
    g.ldslab = g.Qn;
    return (unsigned)(g.ptiles * g.qtiles * g.ksplit);
  };
  const unsigned n = grid(dh, p.big_dh), m = grid(dw, p.big_dw);
  if (!p.big_dh && !p.big_dw) {
    const unsigned n8 = (n + 7) & ~7u;
    hipLaunchKernelGGL(ce_products_kernel, dim3(n8 + m), dim3(256), 0, st, dh, dw, (int)n8);
  } else {
    launch_product<DH>(dh, p.big_dh, n, st);
    MMST_CHECK_LAUNCH();
    launch_product<DW>(dw, p.big_dw, m, st);
  }
  MMST_CHECK_LAUNCH();
  auto lanes = [](const CeGemm& g) -> unsigned {   // workgroups of 256 that join its slabs
    return g.ksplit > 1 ? (unsigned)(((long)g.Pn * (g.Qn / 4) + (g.dbias ? g.Pn : 0) + 255) / 256) : 0u;
  };
  const unsigned a = lanes(dh), b = lanes(dw);
  if (a + b) {
    hipLaunchKernelGGL(ce_slabs_kernel, dim3(a + b), dim3(256), 0, st, dh, dw, a);
    MMST_CHECK_LAUNCH();
  }
  return MMST_OK;
}
template <int MODE> void launch_logits(CeGemm& g, const CePlan& p, char* ws, hipStream_t st) {
  if (p.split_logits > 1) {
    g.ptiles = (g.Pn + 127) / 128;
    g.qtiles = (g.Qn + 127) / 128;
    g.ksplit = p.split_logits;
    g.slab = (float*)(ws + p.slab_logits);
    g.ldslab = (g.Qn + 7) & ~7;
    const dim3 grid(g.ptiles * g.qtiles * g.ksplit);
    hipLaunchKernelGGL((ce_product_kernel<LOGIT_PART, 128, 128, 2, 2, 4>), grid, dim3(256), 0, st, g);
    hipLaunchKernelGGL(ce_join_kernel<MODE>, dim3((g.Qn + 63) / 64, (g.Pn + 15) / 16), dim3(256), 0, st, g);
    return;
  }
  const int b = p.wide ? 160 : p.big ? 256 : 128;
  g.qtiles = (g.Qn + b - 1) / b;
  if constexpr (MODE == LOGIT_STATS)
    if (p.wide) {
      hipLaunchKernelGGL((ce_logits_kernel<MODE, 128, 160, 4, 1>), dim3(2 * TILE_GRID), dim3(256), 0, st, g);
      return;
    }
  if (p.big) hipLaunchKernelGGL((ce_logits_kernel<MODE, 256, 256, 2, 4>), dim3(TILE_GRID), dim3(512), 0, st, g);
  else if (p.few) hipLaunchKernelGGL((ce_logits_kernel<MODE, 128, 128, 2, 2, 4>), dim3(TILE_GRID), dim3(256), 0, st, g);
  else hipLaunchKernelGGL((ce_logits_kernel<MODE, 128, 128, 2, 2>), dim3(2 * TILE_GRID), dim3(256), 0, st, g);
}
template <int MODE> void launch_stream(CeGemm& g, hipStream_t st) {
  hipLaunchKernelGGL((ce_stream_kernel<MODE>), dim3(STREAM_GRID), dim3(256), 0, st, g);
}

}  // namespace

extern "C" {

int mmst_linear_ce_ws(const mmst_linear_ce_args* args, int grad, size_t* bytes) {
  if (!bytes || !sizes_ok(args)) return MMST_ERR_ARG;
  *bytes = plan(args, grad != 0).total;
  return MMST_OK;
}

int mmst_linear_ce(const mmst_linear_ce_args* args, int grad, void* stream) {
  if (!args_ok(args, grad != 0)) return MMST_ERR_ARG;
  const mmst_linear_ce_args& A = *args;
  const CePlan p = plan(args, grad != 0);
  if (A.N == 0 && !grad) return MMST_OK;
  if (!A.ws || (uintptr_t)A.ws % 256 || A.ws_bytes < p.total) return MMST_ERR_ARG;
  hipStream_t st = (hipStream_t)stream;
  char* ws = (char*)A.ws;
  int* count = (int*)ws;
  float* unit = (float*)ws + 1;
  int* index = (int*)(ws + p.index);
  int* words = (int*)(ws + p.words);
  const bf16* w = (const bf16*)A.w;
  const int D = A.D, V = A.V, N = A.N, D8 = D / 8;

  const int pairs = p.pairs;
  CeGemm logit = {};
  logit.Q = w; logit.ldq = A.ldw; logit.Qn = V; logit.K = D; logit.ksplit = 1;
  logit.bias = A.bias; logit.target = A.target;
  logit.part = (float2*)(ws + p.part); logit.tlogit = (float*)(ws + p.tlogit);
  logit.rows_max = (int)p.rows;
  if (!p.number) {
    for (int i = 0; i < p.pieces; ++i) {
      const long row0 = i * p.rows;
      const int rows = (int)(N - row0 < p.rows ? N - row0 : p.rows);
      logit.P = (const bf16*)A.h + row0 * A.ldh; logit.ldp = A.ldh; logit.rows_max = rows; logit.Pn = rows;
      logit.target = A.target + row0;
      if (p.whole) {
        logit.loss_out = A.loss; logit.lse_out = A.lse; logit.ignore = A.ignore_index;
        launch_stream<LOGIT_LOSS>(logit, st);
        MMST_CHECK_LAUNCH();
        return MMST_OK;
      }
      if (p.stream) launch_stream<LOGIT_STATS>(logit, st);
      else launch_logits<LOGIT_STATS>(logit, p, ws, st);
      MMST_CHECK_LAUNCH();
      hipLaunchKernelGGL(ce_rows_kernel, dim3((rows + 15) / 16), dim3(256), 0, st, logit.part, pairs, rows,
                         p.stream ? STREAM_GRID : 0, nullptr, 0, rows, nullptr, logit.target, A.ignore_index, V, logit.tlogit,
                         nullptr, A.loss + row0, A.lse ? A.lse + row0 : nullptr);
      MMST_CHECK_LAUNCH();
    }
    return MMST_OK;
  }

  bf16* hc = (bf16*)(ws + p.hc);
  bf16* gbuf = (bf16*)(ws + p.g);
  float2* lse_c = grad ? (float2*)(ws + p.lse) : nullptr;
  float* weight = grad ? (float*)(ws + p.weight) : nullptr;
  bf16* clear = grad ? (bf16*)A.dh : nullptr;
  const float* dloss = grad ? A.dloss : nullptr;
  const float grad_scale = grad ? A.grad_scale : 1.f;
  const bool merged = p.pieces == 1 && N > 0 && N <= MERGE_ROWS;
  if (merged)
    hipLaunchKernelGGL(ce_index_gather_kernel, dim3((N + 15) / 16), dim3(256), 0, st, (const bf16*)A.h, A.ldh, D8, A.target,
                       A.ignore_index, N, V, dloss, grad_scale, index, words, count, unit, weight, hc, A.loss, A.lse, clear,
                       A.lddh);
  else
    hipLaunchKernelGGL(ce_index_kernel, dim3(1), dim3(1024), 0, st, A.target, A.ignore_index, N, V, index, words, count, A.loss,
                       A.lse, dloss, grad_scale, unit);
  MMST_CHECK_LAUNCH();
  for (int i = 0; i < p.pieces; ++i) {
    const int row0 = (int)(i * p.rows);
    const int rows_max = (int)p.rows;
    const unsigned gather = (unsigned)((p.rows * D8 + 255) / 256);
    if (!merged) {
      hipLaunchKernelGGL(ce_gather_kernel, dim3(gather + (i || !grad ? 0 : (N + 15) / 16)), dim3(256), 0, st, (const bf16*)A.h,
                         A.ldh, D8, index, count, row0, rows_max, dloss, grad_scale, hc, weight, unit, gather, A.target,
                         A.ignore_index, N, V, clear, A.lddh);
      MMST_CHECK_LAUNCH();
    }
    logit.P = hc; logit.ldp = D; logit.Pn = rows_max; logit.count = count; logit.row0 = row0; logit.index = index + row0;
    logit.word = words + row0;
    logit.g = gbuf; logit.ldg = p.Vp;
    if (p.stream) launch_stream<LOGIT_STATS>(logit, st);
    else if (grad) launch_logits<LOGIT_EXP>(logit, p, ws, st);
    else launch_logits<LOGIT_STATS>(logit, p, ws, st);
    MMST_CHECK_LAUNCH();
    logit.lse = lse_c; logit.weight = weight;
    logit.loss_out = A.loss; logit.lse_out = A.lse;
    const dim3 scale((unsigned)((p.Vp + 2047) / 2048 * (p.rows / 4)));
    if (!grad || p.stream || V > JOIN_VOCAB) {
      hipLaunchKernelGGL(ce_rows_kernel, dim3((unsigned)(p.rows / 16)), dim3(256), 0, st, logit.part, pairs, rows_max,
                         p.stream ? STREAM_GRID : 0, count, row0, rows_max, index, A.target, A.ignore_index, V, logit.tlogit,
                         lse_c, A.loss, A.lse);
      MMST_CHECK_LAUNCH();
      if (!grad) continue;
      if (p.stream) launch_stream<LOGIT_GRAD>(logit, st);
      else hipLaunchKernelGGL(ce_scale_kernel<false>, scale, dim3(256), 0, st, logit, pairs);
    } else {
      hipLaunchKernelGGL(ce_scale_kernel<true>, scale, dim3(256), 0, st, logit, pairs);
    }
    MMST_CHECK_LAUNCH();

    CeGemm dh = {};
    dh.P = gbuf; dh.ldp = p.Vp; dh.Pn = rows_max; dh.Q = w; dh.ldq = A.ldw; dh.Qn = D; dh.K = V;
    dh.count = count; dh.row0 = row0; dh.rows_max = rows_max; dh.index = index + row0; dh.ksplit = p.split_dh;
    dh.unit = unit; dh.out = A.dh; dh.ldo = A.lddh; dh.slab = p.split_dh > 1 ? (float*)(ws + p.slab_dh) : nullptr;

    // dw and dbias: in fp32 added to what is there; in bf16 written once, behind sums in fp32 where there are more pieces
    const bool last = i + 1 == p.pieces;
    CeGemm dw = {};
    dw.P = gbuf; dw.ldp = p.Vp; dw.Pn = V; dw.Q = hc; dw.ldq = D; dw.Qn = D;
    dw.count = count; dw.row0 = row0; dw.rows_max = rows_max; dw.ksplit = p.split_dw;
    dw.unit = unit;
    dw.slab = p.split_dw > 1 ? (float*)(ws + p.slab_dw) : nullptr; dw.slab_bias = (float*)(ws + p.slab_bias);
    float* acc = (float*)(ws + p.dwacc);
    dw.ldo = D;
    float* bacc = (float*)(ws + p.dbacc);
    if (dw_f32(&A)) {
      dw.out = A.dw; dw.out_f32 = 1; dw.acc_in = (const float*)A.dw;
    } else {
      dw.out = last ? A.dw : (void*)acc; dw.out_f32 = last ? 0 : 1; dw.acc_in = i > 0 ? acc : nullptr;
    }
    if (A.grad_f32) {
      dw.dbias = A.dbias; dw.dbias_f32 = 1; dw.dbias_in = (const float*)A.dbias;
    } else if (A.dbias) {
      dw.dbias = last ? A.dbias : (void*)bacc; dw.dbias_f32 = last ? 0 : 1; dw.dbias_in = i > 0 ? bacc : nullptr;
    }
    if (launch_products(dh, dw, p, st) != MMST_OK) return MMST_ERR_LAUNCH;
  }
  return MMST_OK;
}

int mmst_sizeof_linear_ce_args(void) { return (int)sizeof(mmst_linear_ce_args); }

}  // extern "C"
