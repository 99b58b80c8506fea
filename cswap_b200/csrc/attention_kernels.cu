// Attention, forward and backward.  With a query row q_i, the keys j it may see, and scale c:
//
//   s_j = c q_i.k_j,  L_i = log sum exp s_j,  p_j = exp(s_j - L_i),  o_i = sum p_j v_j
//   D_i = do_i.o_i,  ds_j = p_j (do_i.v_j - D_i)
//   dq_i = c sum ds_j k_j,  dk_j = c sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i
//
// Only L is kept for backward, which forms the probabilities again.  A row that sees no key has o = 0, L = -inf and
// takes part in no gradient.
//
// All products run on the tensor cores, 128 x 128 scores at a time: tiles of 128 tokens are copied into shared memory
// by TMA (columns behind the head's dimension and rows behind the sequence arrive as zeros, so that any dimension up to
// 64 or 128 runs as that), scores and accumulators lie in tensor memory, and the probabilities, rounded to the operands'
// type, go back to tensor memory over the scores they came from, as the first operand of the second product.  The
// second operand of that product is the tile that is in shared memory anyway, read across its rows.
//
// Three kernels, each with a warp that copies, a warp that issues the products, and warps for the softmax, a thread a row
// or half a row; backward, four more that take the results out:
//   forward   a tile of queries, over the tiles of keys: s, p, o += p v
//   dq        the same rows: s, dp = do v, ds, dq += ds k
//   dkv       a tile of keys, over the tiles of queries of every head that shares them: s and dp transposed,
//             dv += p do, dk += ds q
// dq and dkv each form the scores for themselves: seven products where five would do, but no sums over CTAs, whose
// order would change the result from call to call, and no float32 copy of dq in memory.
//
// What bounds it.  For 128 x 128 scores the tensor cores take 256 clocks a product with heads of 64 and 512 with heads of
// 128, the exponentials 1024 (16 a clock and SM; a quarter of them go by polynomial instead), and the rest of the
// softmax's instructions about as long again.  Each kernel by itself, its inputs cold: heads of 128, 4096 causal tokens,
// 32 heads on 8: forward 122 us (1126 TFLOP/s of the pairs that the mask leaves; a large library product reaches 1634), dq
// 193, dkv 221; the tensor cores are busy 59, 53 and 69 % of the time.  Twenty passes of all three in a row take 514 each at
// 1965 MHz, thousands 600 at the 1640 that the power limit leaves.  Heads of 64, 32 sentences of 128 to 512 tokens,
// 12 heads: forward 45 us, dq 67, dkv 61 (24, 24 and 33 % busy): some 2400 clocks a tile of backward, which the softmax
// warps spend one phase after the other (1250 on exponentials, 450 on gradients, the rest on loads, stores and hand-overs).
//
// Numbers that are not: a NaN or an infinity that a query sees shows in its results as the formulas have it.  What the
// masks hide counts for nothing where it lies behind a sequence, or belongs to a query that sees no key.
//
// That the running maximum is followed only where it grows much, and that a part of the exponentials goes by polynomial,
// are published methods for attention on this generation of tensor cores; range reduction and polynomial are those of any
// exponential (Cody and Waite), the coefficients fitted here.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attention_kernels.h"
#include "hand_over.cuh"
#include "internal.h"
#include "pdl.cuh"
#include "tensor_core.cuh"
#include "values.cuh"
#include "waits.h"

namespace csw {
namespace {

using namespace tc;

constexpr int kTile = 128;                 // tokens of a tile
constexpr uint32_t kChunk = kTile * 128;   // bytes of a tile's 64 columns
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// a tensor that is read by rows
struct View {
  const void* p;
  int64_t b, h, t;
  template <class T>
  __device__ const T* row(int batch, int head, int token) const {
    return static_cast<const T*>(p) + batch * b + head * h + token * t;
  }
};
View view_of(const csw_attention_operand& o) { return {o.data, o.batch_stride, o.head_stride, o.token_stride}; }

struct Shape {
  uint32_t batch, heads, kv_heads, q_len, k_len, dim, share;  // share: query heads of a key head
  int causal;
  bool negate;     // the scale is negative: the products are negated instead
  float scale;     // as given
  float exponent;  // |scale| log2(e), and not zero, so that masked scores stay -inf
  const int32_t* lens;
  long long patience;  // clocks that a wait may last
  bool idle;           // nothing is copied, so that the waits for it run out
  uint32_t* status;    // in host memory; set where a wait ran out
  __device__ int keys(uint32_t b) const { return lens ? min(max(lens[b], 0), (int)k_len) : (int)k_len; }
  // keys that query i sees
  __device__ int limit(int i, int keys) const {
    return causal ? min(keys, max(i + (int)k_len - (int)q_len + 1, 0)) : keys;
  }
};

__device__ __forceinline__ void give_up(uint32_t* flag) { *reinterpret_cast<volatile uint32_t*>(flag) = 1; }
// Leaves the role it stands in; the second form for warps that go on together.
#define CSW_WAIT(bar, parity)                \
  if (!bar_wait(bar, parity, s.patience)) {  \
    give_up(flag);                           \
    return;                                  \
  }
#define CSW_WAIT_WARP(bar, parity)                                         \
  if (!__all_sync(0xffffffffu, bar_wait(bar, parity, s.patience))) {       \
    give_up(flag);                                                         \
    return;                                                                \
  }

template <class T>
constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;

// 32 columns of an accumulator, times f, to columns [at, at + 32) of row `row` of a tile of 64, swizzled as the tile
// copies want it
template <class T>
__device__ __forceinline__ void stage_columns(char* tile, int row, int at, const uint32_t* r, float f) {
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    uint4 v;
    v.x = word_of<T>(__uint_as_float(r[i]) * f, __uint_as_float(r[i + 1]) * f);
    v.y = word_of<T>(__uint_as_float(r[i + 2]) * f, __uint_as_float(r[i + 3]) * f);
    v.z = word_of<T>(__uint_as_float(r[i + 4]) * f, __uint_as_float(r[i + 5]) * f);
    v.w = word_of<T>(__uint_as_float(r[i + 6]) * f, __uint_as_float(r[i + 7]) * f);
    *reinterpret_cast<uint4*>(tile + row * 128 + (((at + i) / 8) ^ (row & 7)) * 16) = v;
  }
}

// All columns of a tile's rows [first, end), zeroed by the warp that issues the products: what lies behind a sequence, or
// belongs to a query that sees nothing, must not meet the zeros of its probabilities as a NaN.
template <int DP>
__device__ __forceinline__ void zero_rows(char* tile, int first, int end = kTile) {
  for (int i = threadIdx.x % 32; i < (end - first) * 8; i += 32)
#pragma unroll
    for (int c = 0; c < DP / 64; ++c)
      *reinterpret_cast<uint4*>(tile + c * kChunk + first * 128 + i * 16) = make_uint4(0, 0, 0, 0);
  async_fence();
  __syncwarp();
}

template <int DP>
__device__ __forceinline__ void copy_tokens(uint32_t dst, const CUtensorMap* map, uint32_t bar, int token, int head,
                                            int batch) {
#pragma unroll
  for (int c = 0; c < DP / 64; ++c) copy_tile(dst + c * kChunk, map, bar, c * 64, token, head, batch);
}
// Tiles are named by their descriptors, read along or across their rows; those of a ring are a step apart.
__device__ __forceinline__ uint64_t along(uint32_t tile) { return tile_desc(tile, 16); }
__device__ __forceinline__ uint64_t across(uint32_t tile) { return tile_desc(tile, kChunk); }
// acc (+)= A B^T: both read along their rows, the reduction over the head's dimension.  Behind the products of a call
// the barriers that are not 0 are arrived at: once these, and all in front, have ended.
template <int DP>
__device__ __forceinline__ void product_rows(uint32_t acc, uint64_t da, uint64_t db, uint32_t desc, uint32_t bar0 = 0,
                                             uint32_t bar1 = 0) {
  if (elected()) {
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
      const uint32_t at = (k / 4 * kChunk + k % 4 * 32) / 16;
      mma(acc, da + at, db + at, desc, k > 0);
    }
    if (bar0) commit(bar0);
    if (bar1) commit(bar1);
  }
}
// acc (+)= P B: P in tensor memory, B read across its rows, the reduction over 128 tokens.  P's first 64 columns lie
// at p, the others at p + half.
__device__ __forceinline__ void product_tokens(uint32_t acc, uint32_t p, uint32_t half, uint64_t db, uint32_t desc,
                                               bool add, uint32_t bar0 = 0, uint32_t bar1 = 0) {
  if (elected()) {
#pragma unroll
    for (int k = 0; k < kTile / 16; ++k)
      mma_tmem(acc, p + k / 4 * half + k % 4 * 8, db + k * (2048 / 16), desc, add || k > 0);
    if (bar0) commit(bar0);
    if (bar1) commit(bar1);
  }
}
__device__ __forceinline__ void commit_to(uint32_t bar) {
  if (elected()) commit(bar);
}

// ---- a CTA's work -----------------------------------------------------------------------------------------------------
// The grid has a CTA for each piece of work (a tile of queries or keys of one head).  One that is done takes over the
// piece of a CTA that has not started, so that copies and products of the next piece begin while the softmax warps still
// write the last one, whatever lengths the sequences have.  The copying warp asks, and tells the others two pieces
// ahead: the piece, -1 at the end, and its sequence's number of keys.
struct Piece {
  int first;         // token, -1: there is no piece
  int keys;          // of its sequence
  int batch, head, kv_head, row;  // row: batch x heads + head, of what is held per row and head
};
struct Work {
  uint4 answer;
  Piece piece[2];
  uint64_t bars[5];  // the answer's; told and read, for each of the two
};
struct WorkBars {
  uint32_t answer, answered, told, read;
  __device__ explicit WorkBars(Work& w)
      : answer(smem_at(&w.answer)), answered(smem_at(w.bars)), told(answered + 8), read(answered + 24) {}
  // one thread, once; `warps` of them listen
  __device__ void init(int warps) const {
    bar_init(answered, 1);
    for (int i = 0; i < 2; ++i) bar_init(told + 8 * i, 1), bar_init(read + 8 * i, warps);
  }
};
// What a warp hears as its i-th piece; false where a wait ran out.
__device__ __forceinline__ bool hear(Work& w, const WorkBars& bars, const Shape& s, int i, Piece* piece) {
  if (!__all_sync(0xffffffffu, bar_wait(bars.told + 8 * (i % 2), i / 2 & 1, s.patience))) return false;
  // one lane's reading: the compiler then knows that all have the same
  const volatile Piece& told = w.piece[i % 2];
  piece->first = __shfl_sync(0xffffffffu, told.first, 0), piece->keys = __shfl_sync(0xffffffffu, told.keys, 0);
  piece->batch = __shfl_sync(0xffffffffu, told.batch, 0), piece->head = __shfl_sync(0xffffffffu, told.head, 0);
  piece->kv_head = __shfl_sync(0xffffffffu, told.kv_head, 0), piece->row = __shfl_sync(0xffffffffu, told.row, 0);
  if (threadIdx.x % 32 == 0) bar_arrive(bars.read + 8 * (i % 2));
  return true;
}

// NaN for all rows of a tensor; a row is a whole number of 16 bytes, and 0x7fff a NaN of either type.
__device__ __noinline__ void spoil(const View& v, uint32_t batch, uint32_t heads, uint32_t tokens, uint32_t dim) {
  const uint32_t packs = dim / 8;
  const uint64_t n = (uint64_t)batch * heads * tokens * packs;
  for (uint64_t i = threadIdx.x; i < n; i += blockDim.x) {
    const uint64_t row = i / packs, head = row / tokens;
    uint4* to = const_cast<uint4*>(reinterpret_cast<const uint4*>(v.row<uint16_t>(head / heads, head % heads, row % tokens)));
    to[i % packs] = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
  }
}
__device__ __noinline__ void spoil(float* p, uint64_t n) {
  for (uint64_t i = threadIdx.x; i < n; i += blockDim.x) p[i] = NAN;
}
// What every kernel ends with, also where a wait ran out: copies on their way get time to land, then spoil() makes all
// results NaN, those of other CTAs that are done as well (which pieces this one still owed no single warp knows); tensor
// memory is freed.
template <int COLUMNS, class F>
__device__ __forceinline__ void leave(const Shape& s, uint32_t* flag, uint32_t tmem, bool owner, F&& spoil) {
  __syncwarp();
  fence_before();
  __syncthreads();
  fence_after();
  if (*reinterpret_cast<volatile uint32_t*>(flag)) {
    for (int i = 0; i < 1000; ++i) __nanosleep(10000);
    spoil();
    if (threadIdx.x == 0) {
      *reinterpret_cast<volatile uint32_t*>(s.status) = 1;
      __threadfence_system();
    }
  }
  if (owner) tmem_free<COLUMNS>(tmem);
}

// The copying warp's lane over all its pieces: f.piece(index) says which one a CTA has, f.copy(piece) copies what it
// needs, and returns false where a wait ran out.
template <class F>
__device__ __forceinline__ void give_work(Work& w, const WorkBars& bars, const Shape& s, uint32_t* flag, F&& f) {
  int index = blockIdx.x;
  for (int i = 0;; ++i) {
    if (i >= 2) CSW_WAIT(bars.read + 8 * (i % 2), (i / 2 - 1) & 1);
    Piece piece{-1};
    if (index >= 0) piece = f.piece(index);
    w.piece[i % 2] = piece;
    bar_arrive(bars.told + 8 * (i % 2));
    if (index < 0) return;
    if (s.idle || !f.copy(piece)) {
      give_up(flag);
      return;
    }
    // Not earlier: a piece that is taken waits until this one is done, however long that is.
    bar_expect(bars.answered, 16);
    take_next(bars.answer, bars.answered);
    CSW_WAIT(bars.answered, i & 1);
    index = taken_index(bars.answer);
    async_fence();  // the answer is read before the next one is written
  }
}

// Tiles of 64 columns are staged by a group of warps, of which one thread, `first`, stores them.  Both are false where a
// wait ran out.
__device__ __forceinline__ bool stage_free(bool first, Meeting& group) {
  if (first) stores_read();
  return group();
}
__device__ __forceinline__ bool stage_full(Meeting& group) {
  async_fence();
  return group();
}

// ---- forward --------------------------------------------------------------------------------------------------------
struct Forward {
  CUtensorMap q, k, v, o;
  Shape s;
  float* lse;
  View out;  // o once more
};

// NWG tiles of 128 queries a CTA; columns of tensor memory: the scores of each, then the sums of each.  Shared memory:
// the queries, a ring of key and value tiles, and 64 columns of results of each.
template <int DP, int NWG>
struct ForwardPlan {
  static constexpr int kThreads = NWG * 128 + 64;
  static constexpr uint32_t kTileBytes = kTile * DP * 2;
  static constexpr int kStages = 4;
  static constexpr size_t kShared = (NWG + kStages) * kTileBytes + NWG * kChunk;
  static constexpr int kColumns = NWG * (128 + DP) > 256 ? 512 : 256;
};

// Piece `index` of a grid over `tokens` queries a CTA.  The last ones of a causal mask see the most keys: they go first.
__device__ __forceinline__ Piece piece_of_queries(const Shape& s, int index, int tokens) {
  const int per = s.batch * s.heads, tiles = gridDim.x / per, row = index % per, b = row / s.heads, h = row % s.heads;
  return {(tiles - 1 - index / per) * tokens, s.keys(b), b, h, h / (int)s.share, row};
}
template <int NWG>
struct Queries {
  int count[NWG], most;  // tiles of keys that each tile of queries sees
  __device__ Queries(const Shape& s, const Piece& p) {
    most = 0;
#pragma unroll
    for (int w = 0; w < NWG; ++w) {
      const int first = p.first + w * kTile;
      count[w] = first < (int)s.q_len ? (s.limit(min(first + kTile, (int)s.q_len) - 1, p.keys) + kTile - 1) / kTile : 0;
      most = max(most, count[w]);
    }
  }
};

// A thread's row of 128 scores in tensor memory, 32 columns at a time, twice: the largest score, then the exponentials,
// which go over the scores, and their sum.  MASKED: only the first `chunks` chunks of 32 are seen by any row of the warp,
// and this row sees `end` columns.
__device__ __forceinline__ void top_of(float (&m)[4], const uint32_t* r) {
#pragma unroll
  for (int i = 0; i < 32; i += 8)
#pragma unroll
    for (int c = 0; c < 4; ++c) m[c] = max3(m[c], __uint_as_float(r[i + 2 * c]), __uint_as_float(r[i + 2 * c + 1]));
  settle(m[0], m[1], m[2], m[3]);
}
template <bool MASKED>
__device__ __forceinline__ float row_top(uint32_t at, int chunks, int end) {
  float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  if (MASKED) {
#pragma unroll 1
    for (int q = 0; q < chunks; ++q, end -= 32) {
      uint32_t r[32];
      load32(at + 32 * q, r);
      wait_loads(r);
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (i >= end) r[i] = 0xff800000u;
      top_of(m, r);
    }
  } else {
    uint32_t r[2][32];
    load32(at, r[0]);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      wait_loads(r[q % 2]);
      if (q < 3) load32(at + 32 * (q + 1), r[(q + 1) % 2]);
      top_of(m, r[q % 2]);
    }
  }
  return max2(max3(m[0], m[1], m[2]), m[3]);
}
template <class T>
__device__ __forceinline__ void exp_of(Pair (&add)[2], const uint32_t* r, float exponent, float shift, int end,
                                       uint32_t* p) {
  const Pair by = {exponent, exponent}, less = {-shift, -shift};
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    Pair x = fma2({__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])}, by, less);
    // One pair in four by polynomial: the unit for exponentials takes 8 clocks for a warp's, more than all else of a value.
    if (i % 4 == 3) {
      x = exp2_poly(x);
    } else {
      x.x = exp2_fast(x.x), x.y = exp2_fast(x.y);
    }
    if (2 * i >= end) x.x = 0.0f;
    if (2 * i + 1 >= end) x.y = 0.0f;
    add[i % 2] = add2(add[i % 2], x);
    p[i] = word_of<T>(x.x, x.y);
  }
  settle(add[0].x, add[0].y, add[1].x, add[1].y);
}
template <class T, bool MASKED>
__device__ __forceinline__ float row_exp(uint32_t at, int chunks, int end, float exponent, float shift) {
  Pair add[2] = {};
  if (MASKED) {
#pragma unroll 1
    for (int q = 0; q < 4; ++q, end -= 32) {
      uint32_t p[16];
      if (q < chunks) {
        uint32_t r[32];
        load32(at + 32 * q, r);
        wait_loads(r);
        exp_of<T>(add, r, exponent, shift, end, p);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) p[i] = 0;
      }
      store16(at + 16 * q, p);
    }
  } else {
    uint32_t r[2][32];
    load32(at, r[0]);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t p[16];
      wait_loads(r[q % 2]);
      if (q < 3) load32(at + 32 * (q + 1), r[(q + 1) % 2]);
      exp_of<T>(add, r[q % 2], exponent, shift, 32, p);
      store16(at + 16 * q, p);
    }
  }
  return (add[0].x + add[0].y) + (add[1].x + add[1].y);
}

template <class T, int DP, int NWG>
__global__ void __launch_bounds__(ForwardPlan<DP, NWG>::kThreads, NWG == 1 ? 2 : 1)
    attention_forward_kernel(const __grid_constant__ Forward a) {
  using Plan = ForwardPlan<DP, NWG>;
  extern __shared__ __align__(1024) char tiles[];  // the swizzle goes by addresses
  __shared__ Work work;
  __shared__ uint64_t bars[2 + 2 * Plan::kStages + 5 * NWG];
  __shared__ uint32_t tmem_at, flag_word;
  const uint32_t tiles_at = smem_at(tiles);
  const WorkBars work_bars(work);
  const uint32_t q_full = smem_at(bars), q_empty = q_full + 8, full = q_full + 16, empty = full + 8 * Plan::kStages,
                 s_full = empty + 8 * Plan::kStages, p_ready = s_full + 8 * NWG, o_full = p_ready + 8 * NWG,
                 o_free = o_full + 8 * NWG, meet = o_free + 8 * NWG;
  uint32_t* flag = &flag_word;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0);  // known to be the same in all lanes

  if (threadIdx.x == 0) {
    work_bars.init(1 + 4 * NWG);
    bar_init(q_full, 1), bar_init(q_empty, 1);
    for (int i = 0; i < Plan::kStages; ++i) bar_init(full + 8 * i, 1), bar_init(empty + 8 * i, 1);
    for (int i = 0; i < NWG; ++i) {
      bar_init(s_full + 8 * i, 1), bar_init(p_ready + 8 * i, 128);
      bar_init(o_full + 8 * i, 1), bar_init(o_free + 8 * i, 128), bar_init(meet + 8 * i, 4);
    }
    init_visible();
    flag_word = 0;
  }
  if (warp == 4 * NWG && threadIdx.x % 32 == 0) prefetch_map(&a.q), prefetch_map(&a.k), prefetch_map(&a.v);
  // In front of the allocation: what runs before in the stream may want this SM's tensor memory yet.
  pdl_wait();
  if (warp == 4 * NWG + 1) tmem_alloc<Plan::kColumns>(smem_at(&tmem_at));
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_at;
  const Shape& s = a.s;
  const uint32_t ring = tiles_at + NWG * Plan::kTileBytes;

  if (warp == 4 * NWG) {
    struct Copies {
      const Forward& a;
      uint32_t tiles_at, ring, q_full, q_empty, full, empty;
      int i = 0, u = 0;  // tiles of the ring, pieces with any
      __device__ Piece piece(int index) const { return piece_of_queries(a.s, index, NWG * kTile); }
      __device__ bool copy(const Piece& p) {
        const Queries<NWG> at(a.s, p);
        if (at.most == 0) return true;
        if (u > 0 && !bar_wait(q_empty, (u - 1) & 1, a.s.patience)) return false;
        bar_expect(q_full, NWG * Plan::kTileBytes);
#pragma unroll
        for (int w = 0; w < NWG; ++w)
          copy_tokens<DP>(tiles_at + w * Plan::kTileBytes, &a.q, q_full, p.first + w * kTile, p.head, p.batch);
        for (int j = 0; j < 2 * at.most; ++j, ++i) {  // k 0, v 0, k 1, v 1, ...
          const int stage = i % Plan::kStages;
          if (i >= Plan::kStages && !bar_wait(empty + 8 * stage, (i / Plan::kStages - 1) & 1, a.s.patience)) return false;
          bar_expect(full + 8 * stage, Plan::kTileBytes);
          copy_tokens<DP>(ring + stage * Plan::kTileBytes, j % 2 ? &a.v : &a.k, full + 8 * stage, j / 2 * kTile, p.kv_head, p.batch);
        }
        ++u;
        return true;
      }
    };
    if (threadIdx.x % 32 == 0)
      give_work(work, work_bars, s, flag, Copies{a, tiles_at, ring, q_full, q_empty, full, empty});
  } else if (warp == 4 * NWG + 1) {
    [&] {
      const uint32_t scores = product_desc(kBf16<T>, kTile, false, s.negate);
      const uint32_t sums = product_desc(kBf16<T>, DP, true, false);
      constexpr uint32_t kStep = Plan::kTileBytes / 16;
      const uint64_t q_rows = along(tiles_at), ring_rows = along(ring), ring_tokens = across(ring);
      int base = 0, u = 0, tile[NWG] = {}, done[NWG] = {};  // of the ring; pieces; of each tile of queries: tiles, pieces
      for (int it = 0;; ++it) {
        Piece piece;
        if (!hear(work, work_bars, s, it, &piece)) return give_up(flag);
        if (piece.first < 0) return;
        const Queries<NWG> at(s, piece);
        if (at.most == 0) continue;
        CSW_WAIT_WARP(q_full, u & 1);
        for (int j = 0; j <= at.most; ++j) {
          const int ki = base + 2 * j, vi = ki - 1, k = ki % Plan::kStages, v = vi % Plan::kStages;
          if (j < at.most) CSW_WAIT_WARP(full + 8 * k, ki / Plan::kStages & 1);
          if (j > 0) {
            CSW_WAIT_WARP(full + 8 * v, vi / Plan::kStages & 1);
            if (s.lens && j * kTile > piece.keys)
              zero_rows<DP>(tiles + (NWG + v) * Plan::kTileBytes, piece.keys - (j - 1) * kTile);
          }
#pragma unroll
          for (int w = 0; w < NWG; ++w) {
            const uint32_t sw = tmem + w * 128, ow = tmem + NWG * 128 + w * DP;
            if (j > 0 && j <= at.count[w]) {
              CSW_WAIT_WARP(p_ready + 8 * w, tile[w]++ & 1);
              if (j == 1 && done[w] > 0) CSW_WAIT_WARP(o_free + 8 * w, (done[w] - 1) & 1);
              fence_after();
              const bool last = j == at.count[w];
              product_tokens(ow, sw, 32, ring_tokens + v * kStep, sums, j > 1, last ? o_full + 8 * w : 0);
              done[w] += last;
            }
            if (j < at.count[w]) {
              product_rows<DP>(sw, q_rows + w * kStep, ring_rows + k * kStep, scores, s_full + 8 * w);
            }
          }
          if (j < at.most) commit_to(empty + 8 * k);
          if (j > 0) commit_to(empty + 8 * v);
          if (j + 1 == at.most) commit_to(q_empty);
        }
        base += 2 * at.most, ++u;
      }
    }();
  } else {
    const int w = warp / 4, t = threadIdx.x % 128;
    const uint32_t lanes = (uint32_t)(warp % 4 * 32) << 16;
    const uint32_t sw = tmem + w * 128 + lanes, ow = tmem + NWG * 128 + w * DP + lanes;
    char* stage = tiles + (NWG + Plan::kStages) * Plan::kTileBytes + w * kChunk;
    Meeting group{meet + 8 * w, s.patience};
    [&] {
      int tile = 0, done = 0;
      for (int it = 0;; ++it) {
        Piece piece;
        if (!hear(work, work_bars, s, it, &piece)) return give_up(flag);
        if (piece.first < 0) return;
        const Queries<NWG> at(s, piece);
        const int keys = piece.keys, n = NWG == 1 || w == 0 ? at.count[0] : at.count[NWG - 1];
        const int q0 = piece.first + w * kTile, row = q0 + t;
        const int limit = s.limit(row, keys), least = s.limit(q0, keys);
        float top = -INFINITY, sum = 0.0f;
        for (int j = 0; j < n; ++j) {
          CSW_WAIT_WARP(s_full + 8 * w, tile & 1);
          ++tile;
          fence_after();
          // What the mask leaves out for a whole warp is not looked at.
          const bool masked = (j + 1) * kTile > least;
          const int end = limit - j * kTile;
          const int chunks = masked ? min((s.limit(q0 + warp % 4 * 32 + 31, keys) - j * kTile + 31) / 32, 4) : 4;
          const float now = masked ? row_top<true>(sw, chunks, end) : row_top<false>(sw, 4, 0);
          // The maximum is followed only where it grows by more than 2^8: the sums' exponents have room for that, and
          // so has float16, whose largest number is 2^16.  A NaN is followed as well.
          if (__any_sync(0xffffffffu, !((now - top) * s.exponent <= 8.0f))) {
            const float next = max2(top, now);
            const float f = next == -INFINITY ? 1.0f : exp2_fast((top - next) * s.exponent);
            top = next;
            sum *= f;
            if (j > 0) {
#pragma unroll
              for (int c = 0; c < DP; c += 32) {
                uint32_t o[32];
                load32(ow + c, o);
                wait_loads(o);
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                store32(ow + c, o);
              }
            }
          }
          const float shift = top == -INFINITY ? 0.0f : top * s.exponent;
          sum += masked ? row_exp<T, true>(sw, chunks, end, s.exponent, shift)
                        : row_exp<T, false>(sw, 4, 0, s.exponent, shift);
          wait_stores();
          fence_before();
          bar_arrive(p_ready + 8 * w);
        }
        if (n > 0) {
          CSW_WAIT_WARP(o_full + 8 * w, done & 1);
          ++done;
          fence_after();
        }
        // Whether a row sees any key is told by the mask, not by its sum: scores may be infinite or NaN, and show.
        const bool live = limit > 0;
        const float f = live ? 1.0f / sum : 0.0f;
        if (row < (int)s.q_len)
          a.lse[(uint64_t)piece.row * s.q_len + row] =
              !live ? -INFINITY : top == INFINITY ? INFINITY : (top * s.exponent + log2f(sum)) * kLn2;
#pragma unroll
        for (int c = 0; c < DP; c += 64) {
          if (!stage_free(t == 0, group)) return give_up(flag);
          uint32_t o[64] = {};
          if (n > 0) {
            load32(ow + c, o), load32(ow + c + 32, o + 32);
            wait_loads(o), wait_loads(o + 32);
            if (c + 64 == DP) {
              fence_before();
              bar_arrive(o_free + 8 * w);
            }
          }
          if (!live) {
#pragma unroll
            for (int i = 0; i < 64; ++i) o[i] = 0;
          }
          stage_columns<T>(stage, t, 0, o, f), stage_columns<T>(stage, t, 32, o + 32, f);
          if (!stage_full(group)) return give_up(flag);
          if (t == 0 && q0 < (int)s.q_len) store_tile(&a.o, smem_at(stage), c, q0, piece.head, piece.batch);
        }
      }
    }();
    if (t == 0) stores_read();
  }
  leave<Plan::kColumns>(s, flag, tmem, warp == 4 * NWG + 1, [&] {
    spoil(a.out, s.batch, s.heads, s.q_len, s.dim);
    spoil(a.lse, (uint64_t)s.batch * s.heads * s.q_len);
  });
}

// ---- backward ---------------------------------------------------------------------------------------------------------
// Per head and query, padded to whole tiles, dq leaves for dkv in rows[0] log2(e) L, +inf for a query that sees nothing
// and behind the last one, so that its probabilities are zero, and in rows[1] D.  L itself may be infinite where a row
// sees infinite scores; its probabilities are NaN, as its o is.
struct Backward {
  CUtensorMap q, k, v, dout, dq, dk, dv;
  Shape s;
  View o, grad;  // o and do once more, read by rows
  const float* lse;
  float* rows;
  uint32_t padded;
  // dkv, where there are fewer tiles of keys than SMs: the tiles of queries are split into `parts`, whose sums (float32, for
  // each part, key head, key of a whole tile: dv, then dk) a launch of its own adds up
  int parts;
  float* sums;
  uint32_t k_padded;
  View dq_out, dk_out, dv_out;  // the results once more
};

// Both kernels: 256 threads for the scores (two a row, 64 columns each), 128 that prepare a piece's rows and take its
// results out of tensor memory, so that the first ones go from piece to piece without a pause, a warp that copies and
// one for the products.  Tensor memory: a tile for s, one for dp, then the sums.  Shared memory: two tiles that stay for a
// piece, a ring of the others, each with its own barriers, and twice 64 columns of results.
template <int DP>
struct BackwardPlan {
  static constexpr int kThreads = 256 + 128 + 64, kListeners = 13;
  static constexpr uint32_t kTileBytes = kTile * DP * 2;
  static constexpr int kRing = DP == 64 ? 6 : 4, kStay = DP == 64 ? 2 : 1;  // tiles; pieces whose own tiles have a place
  static constexpr size_t kShared = (2 * kStay + kRing) * kTileBytes + 2 * kChunk;
  static constexpr int kColumns = 512;
};

// D = do.o carries the rounding of o, 2^-9 or 2^-12 of it.  sum ds, which would be zero, is what D is off by (r), and is
// put right in dkv's D.  dq would have to lose r sum p k: where a tile of queries sees no more than this many tiles of
// keys that sum is formed too, by a product of its own.  In rows that see more keys o is smaller, by the square root of
// their number, and with it r: of dq's error, 0.0024 of its norm in bfloat16 (ds and dq are rounded), r made up a
// thirtieth at 2048 causal keys, but more than half of 0.0038 at 40.
constexpr int kFewTiles = 2;

// The probabilities of columns k and k + 1.  One pair in four by polynomial: the unit for exponentials takes 8 clocks for
// a warp's, a thousand for a tile's, and the softmax warps have little else to do meanwhile.
__device__ __forceinline__ void exp_pair(int k, const uint32_t* r, Pair by, Pair less, float* p) {
  Pair x = fma2({__uint_as_float(r[k]), __uint_as_float(r[k + 1])}, by, less);
  if (k % 8 == 6) {
    x = exp2_poly(x);
  } else {
    x.x = exp2_fast(x.x), x.y = exp2_fast(x.y);
  }
  p[k] = x.x, p[k + 1] = x.y;
}

// ds = p (dp - D) for 32 columns, rounded and packed over the dp that it came from; their sum
template <class T>
__device__ __forceinline__ float to_gradients(const float* p, const uint32_t* dp, const float* d, uint32_t* out) {
  float sum[2] = {};
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float x = p[2 * i] * (__uint_as_float(dp[2 * i]) - d[2 * i]);
    const float y = p[2 * i + 1] * (__uint_as_float(dp[2 * i + 1]) - d[2 * i + 1]);
    sum[0] += x, sum[1] += y;
    out[i] = word_of<T>(x, y);
  }
  return sum[0] + sum[1];
}

// 64 columns of an accumulator, a thread a row, to a staged tile, or zeros; loaded(): they have left tensor memory
template <class T, class F>
__device__ __forceinline__ void take_columns(char* stage, int t, bool any, bool live, uint32_t at, float f, F&& loaded) {
  uint32_t r[64] = {};
  if (any) {
    load32(at, r), load32(at + 32, r + 32);
    wait_loads(r), wait_loads(r + 32);
    loaded();
  }
  if (!live) {
#pragma unroll
    for (int k = 0; k < 64; ++k) r[k] = 0;
  }
  stage_columns<T>(stage, t, 0, r, f), stage_columns<T>(stage, t, 32, r + 32, f);
}

template <class T, int DP>
__global__ void __launch_bounds__(BackwardPlan<DP>::kThreads, 1) attention_dq_kernel(const __grid_constant__ Backward a) {
  using Plan = BackwardPlan<DP>;
  constexpr int kRing = Plan::kRing, kStay = Plan::kStay;
  extern __shared__ __align__(1024) char tiles[];  // the swizzle goes by addresses
  __shared__ Work work;
  __shared__ uint64_t bars[8 + 2 * kStay + 2 * kRing + 4];
  __shared__ float shifts[2][kTile], deltas[2][kTile];  // of this piece and the next
  __shared__ uint32_t tmem_at, flag_word;
  const uint32_t tiles_at = smem_at(tiles);
  const WorkBars work_bars(work);
  const uint32_t dq_full = smem_at(bars), dq_free = dq_full + 8, q_full = dq_full + 64, q_empty = q_full + 8 * kStay, full = q_empty + 8 * kStay, empty = full + 8 * kRing,
                 s_full = empty + 8 * kRing, s_free = s_full + 8, dp_full = s_free + 8, ds_ready = dp_full + 8;
  // The next piece's rows are ready before the softmax warps have to have looked at this one's, and their sums may be
  // ready before this one's are looked at.
  const Turns rows_ready{dq_full + 16}, left_ready{dq_full + 32};
  const uint32_t meet_results = dq_full + 48, meet_softmax = dq_full + 56;
  uint32_t* flag = &flag_word;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0);  // known to be the same in all lanes
  if (threadIdx.x == 0) {
    work_bars.init(Plan::kListeners);
    bar_init(dq_full, 1), bar_init(dq_free, 128);
    for (int i = 0; i < kStay; ++i) bar_init(q_full + 8 * i, 1), bar_init(q_empty + 8 * i, 1);
    for (int i = 0; i < 2; ++i) bar_init(rows_ready.bar(i), 128), bar_init(left_ready.bar(i), 256);
    bar_init(meet_results, 4), bar_init(meet_softmax, 8);
    for (int i = 0; i < kRing; ++i) bar_init(full + 8 * i, 1), bar_init(empty + 8 * i, 1);
    bar_init(s_full, 1), bar_init(s_free, 256), bar_init(dp_full, 1), bar_init(ds_ready, 256);
    init_visible();
    flag_word = 0;
  }
  if (warp == 12 && threadIdx.x % 32 == 0) prefetch_map(&a.q), prefetch_map(&a.dout), prefetch_map(&a.k), prefetch_map(&a.v);
  // In front of the allocation: what runs before in the stream may want this SM's tensor memory yet.
  pdl_wait();
  if (warp == 13) tmem_alloc<Plan::kColumns>(smem_at(&tmem_at));
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_at, s_at = tmem, dp_at = tmem + 128, dq_at = tmem + 256,
                 pk_at = dq_at + DP;  // sum p k
  const Shape& s = a.s;
  const uint32_t ring = tiles_at + 2 * kStay * Plan::kTileBytes;  // behind q and do: k 0, v 0, k 1, v 1, ...

  if (warp == 12) {
    struct Copies {
      const Backward& a;
      uint32_t tiles_at, ring, q_full, q_empty, full, empty;
      int i = 0, u = 0;  // tiles of the ring, pieces with any
      __device__ Piece piece(int index) const { return piece_of_queries(a.s, index, kTile); }
      __device__ bool copy(const Piece& p) {
        const Queries<1> at(a.s, p);
        if (at.most == 0) return true;
        const uint32_t to = tiles_at + u % kStay * 2 * Plan::kTileBytes, here = q_full + 8 * (u % kStay);
        if (u >= kStay && !bar_wait(q_empty + 8 * (u % kStay), (u / kStay - 1) & 1, a.s.patience)) return false;
        bar_expect(here, 2 * Plan::kTileBytes);
        copy_tokens<DP>(to, &a.q, here, p.first, p.head, p.batch);
        copy_tokens<DP>(to + Plan::kTileBytes, &a.dout, here, p.first, p.head, p.batch);
        for (int j = 0; j < 2 * at.most; ++j, ++i) {
          const int slot = i % kRing;
          if (i >= kRing && !bar_wait(empty + 8 * slot, (i / kRing - 1) & 1, a.s.patience)) return false;
          bar_expect(full + 8 * slot, Plan::kTileBytes);
          copy_tokens<DP>(ring + slot * Plan::kTileBytes, j % 2 ? &a.v : &a.k, full + 8 * slot, j / 2 * kTile, p.kv_head, p.batch);
        }
        ++u;
        return true;
      }
    };
    if (threadIdx.x % 32 == 0)
      give_work(work, work_bars, s, flag, Copies{a, tiles_at, ring, q_full, q_empty, full, empty});
  } else if (warp == 13) {
    [&] {
      const uint32_t scores = product_desc(kBf16<T>, kTile, false, s.negate);
      const uint32_t slopes = product_desc(kBf16<T>, kTile, false, false);
      const uint32_t sums = product_desc(kBf16<T>, DP, true, false);
      // The scores of the next tile come in front of what follows of this one: their place is free once they have been
      // read, that of dp behind the product that reads it.
      constexpr uint32_t kStep = Plan::kTileBytes / 16;
      const uint64_t stay_rows = along(tiles_at), ring_rows = along(ring), ring_tokens = across(ring);
      uint32_t i = 0, u = 0, slot = 0, round = 0;  // tiles of keys, pieces with any; of the ring
      for (int it = 0;; ++it) {
        Piece piece;
        if (!hear(work, work_bars, s, it, &piece)) return give_up(flag);
        if (piece.first < 0) return;
        const int n = Queries<1>(s, piece).most;
        if (n == 0) continue;
        const bool few = n <= kFewTiles;
        const uint32_t stay = u % kStay;
        const uint64_t q_rows = stay_rows + stay * 2 * kStep;  // do behind it
        CSW_WAIT_WARP(q_full + 8 * stay, u / kStay & 1);
        uint32_t before = 0;  // the slot of this turn's tile, whose scores came the turn before
        for (int j = -1; j < n; ++j) {
          const bool now = j >= 0, next = j + 1 < n;
          const uint64_t k_rows = ring_rows + slot * kStep, k_now = ring_tokens + before * kStep;
          if (j == 0 && u > 0) CSW_WAIT_WARP(dq_free, (u - 1) & 1);
          if (now && few) {
            CSW_WAIT_WARP(s_free, (i - 1) & 1);  // the probabilities are there
            fence_after();
            product_tokens(pk_at, s_at, 64, k_now, sums, j > 0);
          }
          if (next) {
            CSW_WAIT_WARP(full + 8 * slot, round & 1);
            if (s.lens && (j + 2) * kTile > piece.keys) {
              const int keys = piece.keys - (j + 1) * kTile;
              zero_rows<DP>(tiles + (2 * kStay + slot) * Plan::kTileBytes, keys);
              CSW_WAIT_WARP(full + 8 * slot + 8, round & 1);
              zero_rows<DP>(tiles + (2 * kStay + slot + 1) * Plan::kTileBytes, keys);
            }
            if (i > 0) CSW_WAIT_WARP(s_free, (i - 1) & 1);
            fence_after();
            product_rows<DP>(s_at, q_rows, k_rows, scores, s_full);
          }
          if (now) {
            CSW_WAIT_WARP(ds_ready, (i - 1) & 1);
            fence_after();
            product_tokens(dq_at, dp_at, 64, k_now, sums, j > 0, empty + 8 * before, !next ? dq_full : 0);
          }
          if (next) {
            CSW_WAIT_WARP(full + 8 * slot + 8, round & 1);
            product_rows<DP>(dp_at, q_rows + kStep, k_rows + kStep, slopes, dp_full, empty + 8 * slot + 8);
          }
          if (j + 2 == n) commit_to(q_empty + 8 * stay);
          before = slot;
          if (next) {
            ++i;
            slot += 2;
            if (slot == kRing) slot = 0, ++round;
          }
        }
        ++u;
      }
    }();
  } else if (warp >= 8) {
    const int t = threadIdx.x - 256;
    const uint32_t lanes = (uint32_t)(warp % 4 * 32) << 16;
    char* stage = tiles + (2 * kStay + kRing) * Plan::kTileBytes;
    Meeting group{meet_results, s.patience};
    // D of the piece's rows, DP / 8 lanes a row; they are read before the next piece's results are waited for.  False
    // where a wait ran out, as below.
    float shift = INFINITY, delta = 0.0f;  // of this thread's row of the piece that was prepared last
    auto prepare = [&](const Piece& p, int u) -> bool {
      const int own = p.first + t;
      const float lse = own < (int)s.q_len ? a.lse[(uint64_t)p.row * s.q_len + own] : 0.0f;
      constexpr int kLanes = DP / 8, kRows = 32 / kLanes, kAtOnce = 8;
      const int lane = t % kLanes, mine = t / 32 * 32 + t % 32 / kLanes;
#pragma unroll
      for (int i = 0; i < 32 / kRows; i += kAtOnce) {
        uint4 x[kAtOnce], y[kAtOnce];  // all loads before the first use: they take some 1000 clocks each
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
          // rows behind the last one stand for that, and are not used
          const int row = min(p.first + mine + (i + k) * kRows, (int)s.q_len - 1);
          x[k] = y[k] = make_uint4(0, 0, 0, 0);
          if (lane * 8 < (int)s.dim) {
            x[k] = *reinterpret_cast<const uint4*>(a.o.row<T>(p.batch, p.head, row) + lane * 8);
            y[k] = *reinterpret_cast<const uint4*>(a.grad.row<T>(p.batch, p.head, row) + lane * 8);
          }
        }
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
          float f[8], g[8], d = 0.0f;
          load_pack(reinterpret_cast<const T*>(&x[k]), f);
          load_pack(reinterpret_cast<const T*>(&y[k]), g);
#pragma unroll
          for (int c = 0; c < 8; ++c) d += f[c] * g[c];
#pragma unroll
          for (int c = kLanes / 2; c; c /= 2) d += __shfl_xor_sync(0xffffffffu, d, c);
          if (lane == 0) deltas[u & 1][mine + (i + k) * kRows] = d;
        }
      }
      // +inf for rows that see nothing alone: probabilities that an infinite L stands for are NaN
      shift = fabsf(lse) == INFINITY ? NAN : lse * kLog2e;
      if (own >= (int)s.q_len || s.limit(own, p.keys) <= 0) shift = INFINITY;
      shifts[u & 1][t] = shift;
      if (!group()) return false;
      delta = deltas[u & 1][t];
      bar_arrive(rows_ready.bar(u));
      return true;
    };
    // The results of a piece that sees n tiles, and its row's exponent shift and D; false where a wait ran out.
    auto finish = [&](const Piece& p, int n, int u, float shift, float d) -> bool {
      const bool live = shift != INFINITY;
      float off = 0.0f;
      if (n > 0) {
        if (!__all_sync(0xffffffffu, bar_wait(left_ready.bar(u), left_ready.parity(u), s.patience) && bar_wait(dq_full, u & 1, s.patience))) return false;
        fence_after();
        off = live ? shifts[u & 1][t] + deltas[u & 1][t] : 0.0f;
        if (!(fabsf(off) < INFINITY)) off = 0.0f;  // of gradients that are not finite nothing is put right
      }
      if (!stage_free(t == 0, group)) return false;
#pragma unroll
      for (int c = 0; c < DP; c += 32) {
        uint32_t r[32] = {};
        if (n > 0) {
          load32(dq_at + c + lanes, r);
          wait_loads(r);
          if (n <= kFewTiles) {
            uint32_t m[32];
            load32(pk_at + c + lanes, m);
            wait_loads(m);
#pragma unroll
            for (int k = 0; k < 32; ++k) r[k] = __float_as_uint(fmaf(-off, __uint_as_float(m[k]), __uint_as_float(r[k])));
          }
          if (c + 32 == DP) {
            fence_before();
            bar_arrive(dq_free);
          }
        }
        if (!live) {
#pragma unroll
          for (int k = 0; k < 32; ++k) r[k] = 0;
        }
        stage_columns<T>(stage + c / 64 * kChunk, t, c % 64, r, s.scale);
      }
      if (!stage_full(group)) return false;
      if (t == 0) {
#pragma unroll
        for (int c = 0; c < DP; c += 64)
          if (c < (int)s.dim) store_tile(&a.dq, smem_at(stage) + c / 64 * kChunk, c, p.first, p.head, p.batch);
      }
      float* mine = a.rows + (uint64_t)p.row * a.padded + p.first + t;  // padded to whole tiles
      mine[0] = shift;
      mine[(uint64_t)s.batch * s.heads * a.padded] = live ? d + off : 0.0f;
      return true;
    };
    [&] {
      Piece last{-1};
      int last_n = 0, u = 0;
      for (int it = 0;; ++it) {
        Piece piece;
        if (!hear(work, work_bars, s, it, &piece)) return give_up(flag);
        const int n = piece.first >= 0 ? Queries<1>(s, piece).most : 0;
        const float last_shift = shift, last_delta = delta;
        if (n > 0 && !prepare(piece, u)) return give_up(flag);
        if (last.first >= 0 && !finish(last, last_n, u - 1, last_shift, last_delta)) return give_up(flag);
        last.first = -1;
        if (piece.first < 0) return;
        if (n > 0) {
          last = piece, last_n = n;
          ++u;
        } else if (!finish(piece, 0, 0, INFINITY, 0.0f)) {
          return give_up(flag);
        }
      }
    }();
    if (t == 0) stores_read();
  } else {
    const int w = warp / 4, t = threadIdx.x % 128;
    const uint32_t lanes = (uint32_t)(warp % 4 * 32) << 16;
    Meeting group{meet_softmax, s.patience};
    [&] {
      int i = 0, u = 0;
      for (int it = 0;; ++it) {
        Piece piece;
        if (!hear(work, work_bars, s, it, &piece)) return give_up(flag);
        if (piece.first < 0) return;
        const int keys = piece.keys, n = Queries<1>(s, piece).most, row = piece.first + t;
        if (n == 0) continue;
        const int limit = s.limit(row, keys), least = s.limit(piece.first, keys);
        CSW_WAIT_WARP(rows_ready.bar(u), rows_ready.parity(u));
        const float shift = shifts[u & 1][t], d = deltas[u & 1][t];
        if (!group()) return give_up(flag);  // both halves have read: the places are written below
        const bool few = n <= kFewTiles;
        float left = 0.0f;  // sum of ds
        for (int j = 0; j < n; ++j, ++i) {
          CSW_WAIT_WARP(s_full, i & 1);
          fence_after();
          float p[64];
          {
            uint32_t r[64];
            load32(s_at + 64 * w + lanes, r);
            load32(s_at + 64 * w + 32 + lanes, r + 32);
            wait_loads(r), wait_loads(r + 32);
            if (!few) {
              fence_before();
              bar_arrive(s_free);
            }
#pragma unroll
            for (int k = 0; k < 64; k += 2)
              exp_pair(k, r, both(s.exponent), both(-shift), p);
          }
          const bool masked = (j + 1) * kTile > least;
          const int end = limit - j * kTile - 64 * w;
          if (masked) {
#pragma unroll
            for (int k = 0; k < 64; ++k)
              if (k >= end) p[k] = 0.0f;
          }
          if (few) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              uint32_t out[16];
#pragma unroll
              for (int k = 0; k < 16; ++k) out[k] = word_of<T>(p[32 * c + 2 * k], p[32 * c + 2 * k + 1]);
              store16(s_at + 64 * w + 16 * c + lanes, out);
            }
            wait_stores();
            fence_before();
            bar_arrive(s_free);
          }
          CSW_WAIT_WARP(dp_full, i & 1);
          fence_after();
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t r[32], out[16];
            float dd[32];
            load32(dp_at + 64 * w + 32 * c + lanes, r);
            wait_loads(r);
#pragma unroll
            for (int k = 0; k < 32; ++k) dd[k] = d;
            left += to_gradients<T>(p + 32 * c, r, dd, out);
            store16(dp_at + 64 * w + 16 * c + lanes, out);
          }
          wait_stores();
          fence_before();
          bar_arrive(ds_ready);
        }
        (w == 0 ? shifts : deltas)[u & 1][t] = left;
        bar_arrive(left_ready.bar(u));
        ++u;
      }
    }();
  }
  leave<Plan::kColumns>(s, flag, tmem, warp == 13, [&] {
    spoil(a.dq_out, s.batch, s.heads, s.q_len, s.dim);
    spoil(a.rows, 2 * (uint64_t)s.batch * s.heads * a.padded);  // and with them what dkv makes of them
  });
}

// Pieces of the grid over keys.  The first keys of a causal mask are seen by the most queries: they go first.
template <bool SPLIT>
struct Keys {
  int from, tiles, n;  // the first tile of queries that sees any of them; tiles of queries; pairs in all
  int head, q;         // the first pair's: head, counted from the first that shares, and tile of queries
  __device__ Keys(const Shape& s, const Piece& p, int parts) {
    // query i sees key j from i = j - (k_len - q_len) on
    from = s.causal ? max(p.first - ((int)s.k_len - (int)s.q_len), 0) / kTile : 0;
    tiles = ((int)s.q_len + kTile - 1) / kTile;
    const int each = p.first < p.keys ? max(tiles - from, 0) : 0;
    head = 0, q = from, n = each * (int)s.share;
    if (SPLIT && n > 0) {
      const int begin = (int)((int64_t)n * part(p) / parts);
      n = (int)((int64_t)n * (part(p) + 1) / parts) - begin;
      head = begin / each, q = from + begin % each;
    }
  }
  // Split, the part stands above the key head (which is below 65536).
  __device__ static int part(const Piece& p) { return p.kv_head >> 16; }
  __device__ static int kv_head(const Piece& p) { return SPLIT ? p.kv_head & 0xffff : p.kv_head; }
};

template <class T, int DP, bool SPLIT>
__global__ void __launch_bounds__(BackwardPlan<DP>::kThreads, 1) attention_dkv_kernel(const __grid_constant__ Backward a) {
  using Plan = BackwardPlan<DP>;
  constexpr int kRing = Plan::kRing, kStay = Plan::kStay;
  extern __shared__ __align__(1024) char tiles[];  // the swizzle goes by addresses
  __shared__ Work work;
  __shared__ uint64_t bars[3 + 2 * kStay + 2 * kRing + 4];
  __shared__ __align__(16) float rows[kRing][kTile];  // with a tile of q the exponents' shifts, with one of do D
  __shared__ uint32_t tmem_at, flag_word;
  const uint32_t tiles_at = smem_at(tiles), rows_at = smem_at(rows);
  const WorkBars work_bars(work);
  const uint32_t sums_full = smem_at(bars), sums_free = sums_full + 8, kv_full = sums_full + 16,
                 kv_empty = kv_full + 8 * kStay, full = kv_empty + 8 * kStay, empty = full + 8 * kRing, s_full = empty + 8 * kRing, p_ready = s_full + 8,
                 dp_full = p_ready + 8, ds_ready = dp_full + 8, meet = ds_ready + 8;
  uint32_t* flag = &flag_word;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0);  // known to be the same in all lanes
  if (threadIdx.x == 0) {
    work_bars.init(Plan::kListeners);
    bar_init(sums_full, 1), bar_init(sums_free, 128);
    for (int i = 0; i < kStay; ++i) bar_init(kv_full + 8 * i, 1), bar_init(kv_empty + 8 * i, 1);
    for (int i = 0; i < kRing; ++i) bar_init(full + 8 * i, 1), bar_init(empty + 8 * i, 1);
    bar_init(s_full, 1), bar_init(p_ready, 256), bar_init(dp_full, 1), bar_init(ds_ready, 256);
    bar_init(meet, 4);
    init_visible();
    flag_word = 0;
  }
  if (warp == 12 && threadIdx.x % 32 == 0) prefetch_map(&a.q), prefetch_map(&a.dout), prefetch_map(&a.k), prefetch_map(&a.v);
  // In front of the allocation: what runs before in the stream may want this SM's tensor memory yet.
  pdl_wait();
  if (warp == 13) tmem_alloc<Plan::kColumns>(smem_at(&tmem_at));
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_at, s_at = tmem, dp_at = tmem + 128, dv_at = tmem + 256, dk_at = dv_at + DP;
  const Shape& s = a.s;
  const uint32_t ring = tiles_at + 2 * kStay * Plan::kTileBytes;  // behind k and v: q 0, do 0, q 1, do 1, ...

  if (warp == 12) {
    struct Copies {
      const Backward& a;
      uint32_t tiles_at, ring, rows_at, kv_full, kv_empty, full, empty;
      int i = 0, u = 0;
      __device__ Piece piece(int index) const {
        const int per = a.s.batch * a.s.kv_heads, row = index % per, b = row / a.s.kv_heads, g = row % a.s.kv_heads;
        const int head = g * (int)a.s.share;  // the first of those that share
        const int tile = SPLIT ? index / per / a.parts : index / per, part = SPLIT ? index / per % a.parts : 0;
        return {tile * kTile, a.s.keys(b), b, head, part << 16 | g, b * (int)a.s.heads + head};
      }
      __device__ bool copy(const Piece& p) {
        const Keys<SPLIT> at(a.s, p, a.parts);
        const int kv_head = at.kv_head(p);
        if (at.n == 0) return true;
        const uint32_t to = tiles_at + u % kStay * 2 * Plan::kTileBytes, here = kv_full + 8 * (u % kStay);
        if (u >= kStay && !bar_wait(kv_empty + 8 * (u % kStay), (u / kStay - 1) & 1, a.s.patience)) return false;
        bar_expect(here, 2 * Plan::kTileBytes);
        copy_tokens<DP>(to, &a.k, here, p.first, kv_head, p.batch);
        copy_tokens<DP>(to + Plan::kTileBytes, &a.v, here, p.first, kv_head, p.batch);
        const uint64_t plane = (uint64_t)a.s.batch * a.s.heads * a.padded;
        int q = at.q, h = at.head;
        // A tile of do is free, for what the products need, before the softmax warps have read the D that came with it.
        // It is not written earlier all the same: the tile of q in front of it in the ring is waited for first, and that is
        // free behind the product that takes the gradients made with D.
        for (int j = 0; j < 2 * at.n; ++j, ++i) {
          const int slot = i % kRing;
          if (i >= kRing && !bar_wait(empty + 8 * slot, (i / kRing - 1) & 1, a.s.patience)) return false;
          const uint32_t bar = full + 8 * slot;
          bar_expect(bar, Plan::kTileBytes + kTile * 4);
          copy_tokens<DP>(ring + slot * Plan::kTileBytes, j % 2 ? &a.dout : &a.q, bar, q * kTile, p.head + h, p.batch);
          copy_bytes(rows_at + slot * (4 * kTile),
                     a.rows + (j % 2 ? plane : 0) + (uint64_t)(p.row + h) * a.padded + (uint64_t)q * kTile, kTile * 4, bar);
          if (j % 2 && ++q == at.tiles) q = at.from, ++h;
        }
        ++u;
        return true;
      }
    };
    if (threadIdx.x % 32 == 0)
      give_work(work, work_bars, s, flag, Copies{a, tiles_at, ring, rows_at, kv_full, kv_empty, full, empty});
  } else if (warp == 13) {
    [&] {
      const uint32_t scores = product_desc(kBf16<T>, kTile, false, s.negate);
      const uint32_t slopes = product_desc(kBf16<T>, kTile, false, false);
      const uint32_t sums = product_desc(kBf16<T>, DP, true, false);
      // Each place in tensor memory is written again behind the product that reads it.
      constexpr uint32_t kStep = Plan::kTileBytes / 16;
      const uint64_t stay_rows = along(tiles_at), ring_rows = along(ring), ring_tokens = across(ring);
      uint32_t i = 0, u = 0, slot = 0, round = 0;  // tiles of queries, pieces with any; of the ring
      for (int it = 0;; ++it) {
        Piece piece;
        if (!hear(work, work_bars, s, it, &piece)) return give_up(flag);
        if (piece.first < 0) return;
        const Keys<SPLIT> at(s, piece, a.parts);
        const int n = at.n;
        if (n == 0) continue;
        // Queries that a causal mask leaves nothing stand in front of the others, in the first keys' first tile.
        const int dead = s.causal && piece.first == 0 ? (int)s.q_len - (int)s.k_len - at.from * kTile : 0;
        int q = at.q;
        const uint32_t stay = u % kStay;
        const uint64_t k_rows = stay_rows + stay * 2 * kStep;  // v behind it
        CSW_WAIT_WARP(kv_full + 8 * stay, u / kStay & 1);
        uint32_t before = 0;  // the slot of this turn's tile, whose scores came the turn before
        for (int j = -1; j < n; ++j) {
          const bool now = j >= 0, next = j + 1 < n;
          const uint64_t q_rows = ring_rows + slot * kStep, q_now = ring_tokens + before * kStep;  // do behind them
          if (now) {
            CSW_WAIT_WARP(p_ready, (i - 1) & 1);
            if (j == 0 && u > 0) CSW_WAIT_WARP(sums_free, (u - 1) & 1);
            fence_after();
            product_tokens(dv_at, s_at, 64, q_now + kStep, sums, j > 0, empty + 8 * before + 8);
          }
          if (next) {
            CSW_WAIT_WARP(full + 8 * slot, round & 1);
            if (dead > 0 && q == at.from) zero_rows<DP>(tiles + (2 * kStay + slot) * Plan::kTileBytes, 0, dead);
            product_rows<DP>(s_at, k_rows, q_rows, scores, s_full);
          }
          if (now) {
            CSW_WAIT_WARP(ds_ready, (i - 1) & 1);
            fence_after();
            product_tokens(dk_at, dp_at, 64, q_now, sums, j > 0, empty + 8 * before, !next ? sums_full : 0);
          }
          if (next) {
            CSW_WAIT_WARP(full + 8 * slot + 8, round & 1);
            if (dead > 0 && q == at.from) zero_rows<DP>(tiles + (2 * kStay + slot + 1) * Plan::kTileBytes, 0, dead);
            product_rows<DP>(dp_at, k_rows + kStep, q_rows + kStep, slopes, dp_full);
          }
          if (j + 2 == n) commit_to(kv_empty + 8 * stay);
          before = slot;
          if (next) {
            ++i;
            slot += 2;
            if (slot == kRing) slot = 0, ++round;
            if (++q == at.tiles) q = at.from;
          }
        }
        ++u;
      }
    }();
  } else if (warp >= 8) {
    const int t = threadIdx.x - 256;
    const uint32_t lanes = (uint32_t)(warp % 4 * 32) << 16;
    char* stage = tiles + (2 * kStay + kRing) * Plan::kTileBytes;
    Meeting group{meet, s.patience};
    [&] {
      int u = 0;
      for (int it = 0;; ++it) {
        Piece piece;
        if (!hear(work, work_bars, s, it, &piece)) return give_up(flag);
        if (piece.first < 0) return;
        const bool any = Keys<SPLIT>(s, piece, a.parts).n > 0;
        if (any) {
          CSW_WAIT_WARP(sums_full, u & 1);
          ++u;
          fence_after();
        }
        // A key behind its sequence has no gradient, whatever its row of the tile held.
        const bool live = any && piece.first + t < piece.keys;
        if constexpr (SPLIT) {
          const uint64_t heads = (uint64_t)s.batch * s.kv_heads, head = (uint64_t)piece.batch * s.kv_heads + Keys<SPLIT>::kv_head(piece);
          float* to = a.sums + ((Keys<SPLIT>::part(piece) * heads + head) * a.k_padded + piece.first + t) * (2 * DP);
#pragma unroll
          for (int c = 0; c < 2 * DP; c += 32) {  // dv, then dk, as they lie in tensor memory
            uint32_t r[32] = {};
            if (any) {
              load32(dv_at + c + lanes, r);
              wait_loads(r);
            }
#pragma unroll
            for (int k = 0; k < 32; k += 4)
              *reinterpret_cast<uint4*>(to + c + k) =
                  live ? make_uint4(r[k], r[k + 1], r[k + 2], r[k + 3]) : make_uint4(0, 0, 0, 0);
          }
          if (any) {
            fence_before();
            bar_arrive(sums_free);
          }
          continue;
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {  // dv, dk
          const uint32_t from = (x == 0 ? dv_at : dk_at) + lanes;
          if (!stage_free(t == 0, group)) return give_up(flag);
#pragma unroll
          for (int c = 0; c < DP; c += 64)
            take_columns<T>(stage + c / 64 * kChunk, t, any, live, from + c, x == 0 ? 1.0f : s.scale, [&] {
              if (x == 1 && c + 64 == DP) {
                fence_before();
                bar_arrive(sums_free);
              }
            });
          if (!stage_full(group)) return give_up(flag);
          if (t == 0) {
#pragma unroll
            for (int c = 0; c < DP; c += 64)
              if (c < (int)s.dim)
                store_tile(x == 0 ? &a.dv : &a.dk, smem_at(stage) + c / 64 * kChunk, c, piece.first, piece.kv_head, piece.batch);
          }
        }
      }
    }();
    if (t == 0) stores_read();
  } else {
    const int w = warp / 4, t = threadIdx.x % 128;
    const uint32_t lanes = (uint32_t)(warp % 4 * 32) << 16;
    [&] {
      int i = 0;
      for (int it = 0;; ++it) {
        Piece piece;
        if (!hear(work, work_bars, s, it, &piece)) return give_up(flag);
        if (piece.first < 0) return;
        const Keys<SPLIT> at(s, piece, a.parts);
        const int n = at.n, row = piece.first + t, off = (int)s.k_len - (int)s.q_len;
        int q = at.q;
        for (int j = 0; j < n; ++j, ++i) {
          const int slot = 2 * i % kRing;
          const uint32_t parity = 2 * i / kRing & 1;
          CSW_WAIT_WARP(full + 8 * slot, parity);  // the rows' numbers
          CSW_WAIT_WARP(s_full, i & 1);
          fence_after();
          float p[64];
          {
            const float4* shifts = reinterpret_cast<const float4*>(rows[slot] + 64 * w);
            uint32_t r[64];
            load32(s_at + 64 * w + lanes, r);
            load32(s_at + 64 * w + 32 + lanes, r + 32);
            wait_loads(r), wait_loads(r + 32);
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const float4 f = shifts[k];
              exp_pair(4 * k, r, both(s.exponent), {-f.x, -f.y}, p);
              exp_pair(4 * k + 2, r, both(s.exponent), {-f.z, -f.w}, p);
            }
          }
          if (s.causal && piece.first + kTile - 1 - off > q * kTile) {
            const int begin = row - off - q * kTile - 64 * w;  // the first query that sees this key
#pragma unroll
            for (int k = 0; k < 64; ++k)
              if (k < begin) p[k] = 0.0f;
          }
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t out[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) out[k] = word_of<T>(p[32 * c + 2 * k], p[32 * c + 2 * k + 1]);
            store16(s_at + 64 * w + 16 * c + lanes, out);
          }
          wait_stores();
          fence_before();
          bar_arrive(p_ready);

          CSW_WAIT_WARP(full + 8 * slot + 8, parity);
          CSW_WAIT_WARP(dp_full, i & 1);
          fence_after();
          const float4* deltas = reinterpret_cast<const float4*>(rows[slot + 1] + 64 * w);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t r[32], out[16];
            float d[32];
            load32(dp_at + 64 * w + 32 * c + lanes, r);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float4 f = deltas[8 * c + k];
              d[4 * k] = f.x, d[4 * k + 1] = f.y, d[4 * k + 2] = f.z, d[4 * k + 3] = f.w;
            }
            wait_loads(r);
            to_gradients<T>(p + 32 * c, r, d, out);
            store16(dp_at + 64 * w + 16 * c + lanes, out);
          }
          wait_stores();
          fence_before();
          bar_arrive(ds_ready);
          if (++q == at.tiles) q = at.from;
        }
      }
    }();
  }
  leave<Plan::kColumns>(s, flag, tmem, warp == 13, [&] {
    if constexpr (SPLIT) {
      spoil(a.sums, (uint64_t)a.parts * s.batch * s.kv_heads * a.k_padded * (2 * DP));
    } else {
      spoil(a.dk_out, s.batch, s.kv_heads, s.k_len, s.dim);
      spoil(a.dv_out, s.batch, s.kv_heads, s.k_len, s.dim);
    }
  });
}

// The parts' sums, in their order; a thread for 4 columns of a key's dv or dk.
template <class T, int DP>
__global__ void __launch_bounds__(256) attention_sums_kernel(const float* __restrict__ sums, Shape s, int parts,
                                                             uint32_t k_padded, View dk, View dv) {
  pdl_wait(sums);
  constexpr int kEach = 2 * DP / 4;
  const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x, at = i / kEach, head = at / s.k_len;
  const uint32_t key = at % s.k_len, c = i % kEach * 4;
  if (head >= (uint64_t)s.batch * s.kv_heads || c % DP >= s.dim) return;
  const float* from = sums + (head * k_padded + key) * (2 * DP) + c;
  const uint64_t step = (uint64_t)s.batch * s.kv_heads * k_padded * (2 * DP);
  float f[4] = {};
#pragma unroll 4
  for (int p = 0; p < parts; ++p) {
    const float4 v = *reinterpret_cast<const float4*>(from + p * step);
    f[0] += v.x, f[1] += v.y, f[2] += v.z, f[3] += v.w;
  }
  if (c >= DP) {
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] *= s.scale;
  }
  const View& to = c < DP ? dv : dk;
  store_pack(const_cast<T*>(to.row<T>(head / s.kv_heads, head % s.kv_heads, key)) + c % DP, f);
}

// ---- host -------------------------------------------------------------------------------------------------------------
Shape shape_of(const csw_attention_shape& s, uint32_t* status) {
  const float e = fmaxf(fabsf(s.scale) * kLog2e, 0x1p-100f);
  const long long wait = wait_limit();
  return {(uint32_t)s.batch, (uint32_t)s.heads, (uint32_t)s.kv_heads, (uint32_t)s.q_len, (uint32_t)s.k_len,
          (uint32_t)s.dim,   (uint32_t)(s.heads / s.kv_heads), s.causal, s.scale < 0.0f, s.scale, e, s.kv_lens,
          wait < 0 ? -wait : wait, wait < 0, status};
}

// tiles of 128 tokens x 64 columns of an operand
bool map_of(CUtensorMap* map, const csw_attention_operand& o, const csw_attention_shape& s, uint64_t heads, uint64_t tokens) {
  const TileEncoder encode = tile_encoder();
  if (!encode) return false;
  const cuuint64_t dims[4] = {s.dim, tokens, heads, s.batch};
  // the stride of an axis of one step is not looked at, but has to be one
  auto bytes = [](ptrdiff_t stride, uint64_t n) { return n > 1 && stride > 0 ? (cuuint64_t)stride * 2 : (cuuint64_t)16; };
  const cuuint64_t strides[3] = {bytes(o.token_stride, tokens), bytes(o.head_stride, heads), bytes(o.batch_stride, s.batch)};
  const cuuint32_t box[4] = {64, kTile, 1, 1}, steps[4] = {1, 1, 1, 1};
  return encode(map, s.type == CSW_TYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                o.data, dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class A>
cudaError_t run(void (*kernel)(const A), uint64_t grid, int threads, size_t shared, cudaStream_t stream, const A& a) {
  const cudaError_t e = taken(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)shared));
  return e != cudaSuccess ? e : pdl_launch(kernel, (unsigned)grid, threads, shared, stream, a);
}

template <class T, int DP, int NWG>
cudaError_t forward(const Forward& a, const csw_attention_shape& s, cudaStream_t stream) {
  using Plan = ForwardPlan<DP, NWG>;
  const uint64_t grid = (s.q_len + NWG * kTile - 1) / (NWG * kTile) * s.batch * s.heads;
  return run(attention_forward_kernel<T, DP, NWG>, grid, Plan::kThreads, Plan::kShared, stream, a);
}
template <class T>
cudaError_t forward_of(const Forward& a, const csw_attention_shape& s, cudaStream_t stream) {
  return s.dim <= 64 ? forward<T, 64, 1>(a, s, stream) : forward<T, 128, 2>(a, s, stream);
}

template <class T, int DP>
cudaError_t backward(const Backward& a, const csw_attention_shape& s, cudaStream_t stream) {
  using Plan = BackwardPlan<DP>;
  cudaError_t e = cudaSuccess;
  if (s.q_len)
    e = run(attention_dq_kernel<T, DP>, (s.q_len + kTile - 1) / kTile * s.batch * s.heads, Plan::kThreads, Plan::kShared,
            stream, a);
  if (e == cudaSuccess && s.k_len)
    e = run(a.parts > 1 ? attention_dkv_kernel<T, DP, true> : attention_dkv_kernel<T, DP, false>, (s.k_len + kTile - 1) / kTile * s.batch * s.kv_heads * a.parts, Plan::kThreads,
            Plan::kShared, stream, a);
  if (e == cudaSuccess && a.parts > 1) {
    const uint64_t threads = (uint64_t)s.batch * s.kv_heads * s.k_len * (2 * DP / 4);
    e = pdl_launch(attention_sums_kernel<T, DP>, (unsigned)((threads + 255) / 256), 256, 0, stream, (const float*)a.sums,
                   a.s, a.parts, a.k_padded, a.dk_out, a.dv_out);
  }
  return e;
}
template <class T>
cudaError_t backward_of(const Backward& a, const csw_attention_shape& s, cudaStream_t stream) {
  return s.dim <= 64 ? backward<T, 64>(a, s, stream) : backward<T, 128>(a, s, stream);
}

}  // namespace

namespace {
uint64_t whole_tiles(uint64_t n) { return (n + kTile - 1) / kTile * kTile; }
// Parts of dkv's work on a tile of keys: enough for two CTAs an SM where there are fewer tiles than SMs, of two tiles of
// queries at least.  (1892 causal tokens, 4 heads of 80 on one: 15 tiles of keys, each with up to 60 of queries.)
int parts_of(const csw_attention_shape& s) {
  const uint64_t tiles = whole_tiles(s.k_len) / kTile * s.batch * s.kv_heads, sms = sm_count();
  if (tiles == 0 || tiles >= sms) return 1;
  const uint64_t most = whole_tiles(s.q_len) / kTile * (s.heads / s.kv_heads) / 2;
  return (int)std::max<uint64_t>(std::min<uint64_t>({2 * sms / tiles, most, 32}), 1);
}
uint64_t row_values(const csw_attention_shape& s) { return 2 * (uint64_t)s.batch * s.heads * whole_tiles(s.q_len); }
}  // namespace

uint64_t attention_workspace_values(const csw_attention_shape& s) {
  const int parts = parts_of(s);
  const uint64_t sums = parts > 1 ? parts * (uint64_t)s.batch * s.kv_heads * whole_tiles(s.k_len) * 2 * (s.dim <= 64 ? 64 : 128) : 0;
  return row_values(s) + sums;
}

cudaError_t attention_forward_launch(const csw_attention_shape& s, const csw_attention_operand& q,
                                     const csw_attention_operand& k, const csw_attention_operand& v,
                                     const csw_attention_operand& o, float* lse, cudaStream_t stream) {
  if (s.batch == 0 || s.q_len == 0) return cudaSuccess;
  if (const cudaError_t e = bind_context()) return e;
  uint32_t* status;
  if (const cudaError_t e = status_word(&status)) return e;
  Forward a;
  a.s = shape_of(s, status), a.lse = lse, a.out = view_of(o);
  if (!map_of(&a.q, q, s, s.heads, s.q_len) || !map_of(&a.o, o, s, s.heads, s.q_len)) return cudaErrorInvalidValue;
  a.k = a.v = a.q;  // without keys nothing is copied from them
  if (s.k_len && (!map_of(&a.k, k, s, s.kv_heads, s.k_len) || !map_of(&a.v, v, s, s.kv_heads, s.k_len)))
    return cudaErrorInvalidValue;
  return s.type == CSW_TYPE_F16 ? forward_of<__half>(a, s, stream) : forward_of<__nv_bfloat16>(a, s, stream);
}

cudaError_t attention_backward_launch(const csw_attention_shape& s, const AttentionBackward& b, cudaStream_t stream) {
  if (s.batch == 0 || (s.q_len == 0 && s.k_len == 0)) return cudaSuccess;
  if (const cudaError_t e = bind_context()) return e;
  uint32_t* status;
  if (const cudaError_t e = status_word(&status)) return e;
  Backward a;
  a.s = shape_of(s, status);
  a.o = view_of(b.o), a.grad = view_of(b.dout);
  a.lse = b.lse, a.rows = b.workspace, a.padded = (uint32_t)whole_tiles(s.q_len);
  a.parts = parts_of(s), a.sums = b.workspace + row_values(s), a.k_padded = (uint32_t)whole_tiles(s.k_len);
  // of an empty side nothing is copied
  a.q = a.k = a.v = a.dout = a.dq = a.dk = a.dv = CUtensorMap{};
  if (s.q_len && (!map_of(&a.q, b.q, s, s.heads, s.q_len) || !map_of(&a.dout, b.dout, s, s.heads, s.q_len) ||
                  !map_of(&a.dq, b.dq, s, s.heads, s.q_len)))
    return cudaErrorInvalidValue;
  if (s.k_len && (!map_of(&a.k, b.k, s, s.kv_heads, s.k_len) || !map_of(&a.v, b.v, s, s.kv_heads, s.k_len) ||
                  !map_of(&a.dk, b.dk, s, s.kv_heads, s.k_len) || !map_of(&a.dv, b.dv, s, s.kv_heads, s.k_len)))
    return cudaErrorInvalidValue;
  a.dq_out = view_of(b.dq), a.dk_out = view_of(b.dk), a.dv_out = view_of(b.dv);
  return s.type == CSW_TYPE_F16 ? backward_of<__half>(a, s, stream) : backward_of<__nv_bfloat16>(a, s, stream);
}

}  // namespace csw
