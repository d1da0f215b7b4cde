// Low-rank adapters of many requests beside projections that their rows share:
//   y[row] = residual[row] + s B (A x[row]),  A [r][k], B [n][r], s of the row's adapter,
// and for the pair of an MLP y = silu(gate + s B (A x)) * (up + s' B' (A' x)).
//
// The two products hang together by the r inner products of a row, which need all of k before the first of n results can be had. Two launches: the first
// leaves the inner products of a few parts of k in a workspace, the second adds these up, multiplies and adds to the rows. The second starts early where its CTAs
// find room: in passes of up to eight rows they have their weights when the first one ends. Of more rows a CTA of the first takes all registers of its SM, and the second's come after it.
//
// Rows find their adapters among 32 (8, in calls of no more): the rows of one adapter are taken together, and what there is to do for all adapters of such a
// block is dealt to its CTAs on the device, which alone knows it: the first launch by (adapter, 32, 64 or 128 ranks of all matrices, part of k), the second by equal shares of
// the columns, weighted with the ranks that stand behind them.
//
// What bounds it, on a B200 whose copies reach 6.46 TB/s: a single row of rank 16 (0.3 MB of weights) takes 4.0 us, of which 1.0 are two launches that do nothing; eight rows of six
// adapters beside three projections (12.7 MB) 9.0 us, 4.6 times the time of their bytes: each launch is a chain of row -> adapter -> rank and address -> weights and activations -> sum,
// and alone they take 5.6 us, of which the products 1.8, and 6.6, of which adding up, products and columns 2.2.
// With many rows it is the products of the first launch and the rows of the second: 512 rows of rank 64 beside 12288 columns take 35.3 us; alone the first launch takes 13.6, of which the
// products 7.2, and the second 26.5: 6.4 before its columns, 1.8 to add up the parts, 3.3 for products, 15 for the rows (50 MB, 7.8 us at the copies' rate) and weights of six units a warp.
//
// Both products run on the tensor cores as m16n8k16, the weights as the 16 rows of an MMA and the rows of the pass as its 8 columns, so that a single token costs
// a quarter of 32 rows and not all of them. Weights of 16 bits are operands as they lie in memory: the order of the dimension that is summed over is
// free, so a lane takes as many consecutive weights as one load brings, and nothing is converted or staged. What they meet, activations and inner products, is
// cut into operands of their type: three bf16 of eight bits each, which is all of an fp32, or two fp16 of 11 bits each after a power of two that brings the
// largest of a row's values at hand to 2^14 .. 2^15 (what is lost of a value is below 2^-22 of it or, where its second fp16 is subnormal, 2^-39 of the largest). Weights of fp32
// are three bf16 too; of the nine products the three smallest are left out: pieces are cut off, not rounded, so that what is left out is below 2^-21 of the product.
#include <algorithm>
#include <cuda_bf16.h>
#include <type_traits>
#include "adapters.h"
#include "common.cuh"

namespace infdev {
namespace {

constexpr int kChunk = 32;      // activations that a warp multiplies at a time
// Columns that a warp multiplies at a time. 32 keep a lane's four columns in one store, but leave no registers for the sums of 32 rows of a pair or of fp32 weights, which then take their
// weights twice: a pair for 128 rows took 32.4 instead of 30.7 us, 97 rows of fp32 weights 13.2 instead of 9.1; 512 rows of rank 64 36.7 instead of 37.2.
constexpr int kUnit = 16;
constexpr int kOuterWarps = 8;
constexpr int inner_warps(int block) { return block > 1 ? 16 : 8; }
constexpr int kParts = 8;       // parts of k: one of the 256 that k is a multiple of has a chunk for each
constexpr int kInner = 4096;    // inner products that a CTA keeps: 128 ranks of 32 rows, or 512 of eight

// How values of a weight's type are multiplied: pieces of a weight, and of what it meets.
template <class W> struct Format {
  static constexpr bool kHalf = std::is_same<W, __half>::value;
  static constexpr int kWeightPieces = sizeof(W) == 4 ? 3 : 1, kPieces = kHalf ? 2 : 3;
};

// D(16x8, f32) += A(16x16, row) * B(16x8, col), fp16 or bf16
template <bool HALF> __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (HALF)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The next eight bits of a and of b as a pair of bf16, which are taken off them. (Of an infinity, a NaN remains.)
__device__ __forceinline__ uint32_t cut_pair(float& a, float& b) {
  const uint32_t hi = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
  a -= __uint_as_float(__float_as_uint(a) & 0xffff0000u), b -= __uint_as_float(__float_as_uint(b) & 0xffff0000u);
  return hi;
}

// Four consecutive values as pieces of a weight's type: word[piece] of the first two, then of the last two.
template <class W> __device__ __forceinline__ void cut_four(float4 v, uint2 (&piece)[Format<W>::kPieces]) {
  if constexpr (Format<W>::kHalf) {
    const uint2 hi = make_uint2(pack_half2(v.x, v.y), pack_half2(v.z, v.w));
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&hi.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi.y));
    piece[0] = hi, piece[1] = make_uint2(pack_half2(v.x - a.x, v.y - a.y), pack_half2(v.z - b.x, v.w - b.y));
  } else {
#pragma unroll
    for (int i = 0; i < Format<W>::kPieces; ++i) {
      piece[i].x = cut_pair(v.x, v.y);
      piece[i].y = cut_pair(v.z, v.w);
    }
  }
}

// The power of two that brings values up to `largest` below 2^15, and its reciprocal; 1 where there is none or they are not finite.
__device__ __forceinline__ void range_of(float largest, float& to, float& back) {
  to = back = 1.f;
  if (largest > 0.f && largest < INFINITY) {
    const uint32_t exponent = min(253u, 268u - (__float_as_uint(largest) >> 23));
    to = __uint_as_float(exponent << 23), back = __uint_as_float((254u - exponent) << 23);
  }
}

// COUNT consecutive weights as they lie in memory. Loads stand apart from what is made of them, so that a batch of loads is under way at once.
template <class W, int COUNT> struct Raw {
  uint32_t word[COUNT * sizeof(W) / 4];
};
// VEC: from lies on a 16-byte boundary; else single weights. (Chosen at run time, a load is issued both ways, one of them with nobody taking part: 16 loads and what packs
// their results for two.)
template <bool VEC, class W> __device__ __forceinline__ void load_raw(Raw<W, 8>& to, const W* from) {
  constexpr int kWords = 8 * sizeof(W) / 4;
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < kWords; i += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(from) + i);
      to.word[i] = v.x, to.word[i + 1] = v.y, to.word[i + 2] = v.z, to.word[i + 3] = v.w;
    }
  } else if constexpr (sizeof(W) == 4) {
#pragma unroll
    for (int i = 0; i < kWords; ++i)
      to.word[i] = __float_as_uint(from[i]);
  } else {
    const uint16_t* half = reinterpret_cast<const uint16_t*>(from);
#pragma unroll
    for (int i = 0; i < kWords; ++i)
      to.word[i] = uint32_t(half[2 * i]) | uint32_t(half[2 * i + 1]) << 16;
  }
}
// Their pieces, two weights a word.
template <class W, int COUNT> __device__ __forceinline__ void pieces_of(const Raw<W, COUNT>& raw, uint32_t (&piece)[Format<W>::kWeightPieces][COUNT / 2]) {
#pragma unroll
  for (int i = 0; i < COUNT / 2; ++i) {
    if constexpr (sizeof(W) == 4) {
      float a = __uint_as_float(raw.word[2 * i]), b = __uint_as_float(raw.word[2 * i + 1]);
#pragma unroll
      for (int w = 0; w < 3; ++w)
        piece[w][i] = cut_pair(a, b);
    } else {
      piece[0][i] = raw.word[i];
    }
  }
}
// d[i] += 16 rows of weights (two consecutive words of `upper` for rows 0 .. 7, of `lower` for 8 .. 15) * eight columns, a sum for each order of magnitude of the
// products: what is added to a sum waits for what was added before, 20 cycles.
template <class W, int WORDS>
__device__ __forceinline__ void add_product(float (&d)[Format<W>::kPieces][4], const uint32_t (&upper)[Format<W>::kWeightPieces][WORDS],
                                            const uint32_t (&lower)[Format<W>::kWeightPieces][WORDS], int at, const uint2 (&column)[Format<W>::kPieces]) {
#pragma unroll
  for (int w = Format<W>::kWeightPieces - 1; w >= 0; --w)
#pragma unroll
    for (int order = Format<W>::kPieces - 1; order >= 0; --order)
      if (order - w >= 0)
        mma<Format<W>::kHalf>(d[order], upper[w][at], lower[w][at], upper[w][at + 1], lower[w][at + 1], column[order - w].x, column[order - w].y);
}
template <int PIECES> __device__ __forceinline__ float total(const float (&d)[PIECES][4], int e) {
  float sum = d[PIECES - 1][e];
#pragma unroll
  for (int i = PIECES - 2; i >= 0; --i)
    sum += d[i][e];
  return sum;
}

// The rows of a block by adapter. Every warp finds out for itself; a lane stands for its row, and for an adapter if its row is the first that has it.
struct Block {
  int base, which;                // the block's first row; the adapter of this lane's row, -1: none
  uint32_t group;                 // the rows of that adapter
  bool leads;
  int rank[kAdapterMaxMatrices];  // of the lane's adapter, 0 where it does not lead
};
template <int ROWS, bool PAIR> __device__ __forceinline__ Block find_block(const AdapterParams& p, int block, bool report) {
  const int lane = threadIdx.x % kWarp;
  Block found;
  found.base = block * ROWS, found.which = -1;
  const int count = min(ROWS, int(p.m) - found.base), matrices = PAIR ? 2 : p.count;
  if (lane < count) {
    const int which = p.rowAdapter[found.base + lane];
    found.which = which >= 0 && which < p.adapterCount ? which : -1;
  }
  found.group = __match_any_sync(0xffffffffu, lane < count ? found.which : -2);
  found.leads = lane < count && __ffs(found.group) - 1 == lane;
#pragma unroll
  for (int i = 0; i < kAdapterMaxMatrices; ++i) {
    uint32_t rank = 0;
    if (found.leads && found.which >= 0 && i < matrices)
      rank = p.adapters[i][found.which].rank;
    if (rank > uint32_t(kAdapterMaxRank)) {
      if (report)
        atomicCAS(p.status, kStatusOk, kStatusBadArgument);  // a wait that was abandoned before, which spoils all rows, stays reported
      rank = 0;
    }
    found.rank[i] = int(rank);
  }
  return found;
}
__device__ __forceinline__ int running_sum(int value) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int other = __shfl_up_sync(0xffffffffu, value, o);
    if (int(threadIdx.x % kWarp) >= o)
      value += other;
  }
  return value;
}
// The rows of `group` in a row, for one warp.
__device__ __forceinline__ void list_rows(int* rows, uint32_t group, int base) {
  const int lane = threadIdx.x % kWarp;
  if (group >> lane & 1)
    rows[__popc(group & ((1u << lane) - 1))] = base + lane;
}

// Inner products between the two launches: [part of k][row of the call][matrix][rank].
template <int BLOCK> __device__ __forceinline__ size_t inner_at(int part, int row, int matrix, int rank) {
  constexpr int kRows = BLOCK > 1 ? kAdapterSlabRows : 8;
  return ((size_t(part) * kRows + row) * kAdapterMaxMatrices + matrix) * kAdapterMaxRank + rank;
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], const void* address) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_u32(address)));
}

// ---- inner products: grid (parts; blocks of 8 BLOCK rows and CTAs of a part and block, which share all items) ----
// An item is some tiles of 16 ranks of an adapter, of all matrices one after the other, some of its rows, and one of kParts parts of k. A part is a sum over chunks of 32
// activations in ascending order, each chunk an MMA sum of its own, so that a row's results do not hang on what it is taken with, but for the way:
//   * up to eight rows: a warp has every eighth chunk, and its activations come as the columns of its MMAs from global memory; the chunks' products meet in shared memory
//   * more: the CTA cuts 128 activations of all rows and brings the weights for them, while those before are multiplied; a warp has a tile, and all chunks
constexpr int kFewTiles = 2, kManyTiles = 8, kRoundChunks = 16, kSpan = 128;
struct InnerShared {
  float result[32][kManyTiles * 16];             // of the CTA's part: [row][rank]
  float parts[kRoundChunks][8][kFewTiles * 16];  // up to eight rows: [chunk][row][rank]
};
template <class W> struct ManyShared {           // more rows
  static constexpr int kAhead = sizeof(W) == 4 ? 1 : Format<W>::kHalf ? 3 : 2;          // spans on their way, as many as there is room for
  static constexpr int kWeightPitch = kSpan * int(sizeof(W)) + 16, kPitch = kSpan + 8;  // 16 bytes more than a multiple of 128: what an MMA's rows have in different banks
  union {
    float result[32][kManyTiles * 16];           // after the last span
    __align__(16) uint8_t weights[kAhead + 1][kManyTiles * 16 * kWeightPitch];
  };
  __align__(16) float uncut[kAhead][32][kSpan];
  __align__(16) uint16_t x[2][Format<W>::kPieces][32][kPitch];
  float back[2][kSpan / kChunk][32];
};

// A tile of ranks of an adapter, counted over all matrices.
template <class W> struct Tile {
  const W* a;  // of the matrix
  int matrix, rank, first;
};
template <class W> __device__ __forceinline__ Tile<W> tile_of(const AdapterParams& p, const int (&rank)[kAdapterMaxMatrices], int adapter, int tile) {
  Tile<W> found{nullptr, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < kAdapterMaxMatrices; ++i) {
    const int here = (rank[i] + 15) / 16;
    if (tile >= 0 && tile < here)
      found.matrix = i, found.rank = rank[i], found.first = tile * 16;
    tile -= here;
  }
  found.a = reinterpret_cast<const W*>(p.adapters[found.matrix][adapter].a);
  return found;
}
// This lane's weights of a tile's 16 rows: rank g, and g + 8 further on (rows past the last are repeated, and their products not used).
template <class W> struct TileRows {
  const W *upper, *lower;
};
template <class W> __device__ __forceinline__ TileRows<W> rows_of(const Tile<W>& tile, int64_t k, int64_t from) {
  const int g = threadIdx.x % kWarp >> 2, t = threadIdx.x & 3;
  const W* const a = tile.a + from + 8 * t;
  return {a + min(tile.first + g, tile.rank - 1) * k, a + min(tile.first + g + 8, tile.rank - 1) * k};
}

template <class W, int BLOCK, bool VEC>
__device__ __forceinline__ void inner_few(const AdapterParams& p, InnerShared& sh, const int (&ranks)[kAdapterMaxMatrices], int adapter, const int* rowsOf, int rows, int firstTile, int tiles,
                                          int part, int chunks, bool& waited) {
  constexpr int kPieces = Format<W>::kPieces, kWeightPieces = Format<W>::kWeightPieces;
  constexpr bool kHalf = Format<W>::kHalf;
  const int tid = threadIdx.x, warp = tid / kWarp, lane = tid % kWarp, g = lane >> 2, t = lane & 3;
  const int64_t from = int64_t(part) * chunks * kChunk;
  TileRows<W> weights[kFewTiles];
#pragma unroll
  for (int i = 0; i < kFewTiles; ++i)
    weights[i] = rows_of(tile_of<W>(p, ranks, adapter, firstTile + min(i, tiles - 1)), p.k, from);
  const float* const x = p.x + int64_t(rowsOf[min(g, rows - 1)]) * p.k + from + 8 * t;  // rows past the last are repeated, and their results not used
  constexpr int kInnerWarps = inner_warps(BLOCK), kThreads = kInnerWarps * kWarp, kOwn = (8 * kFewTiles * 16 + kThreads - 1) / kThreads;
  static_assert(kOwn * kThreads <= 32 * kFewTiles * 16, "rows past the eighth are not read");
  float sum[kOwn] = {};  // of row and rank tid + kThreads i
  Raw<W, 8> next[kFewTiles][2];  // of the chunk after the one at hand
  float4 x0, x1;
  auto load_weights = [&](int c) {
    c = min(c, chunks - 1);
#pragma unroll
    for (int i = 0; i < kFewTiles; ++i) {
      load_raw<VEC>(next[i][0], weights[i].upper + c * kChunk);
      load_raw<VEC>(next[i][1], weights[i].lower + c * kChunk);
    }
  };
  auto load_activations = [&](int c) {
    c = min(c, chunks - 1);
    x0 = *reinterpret_cast<const float4*>(x + c * kChunk), x1 = *reinterpret_cast<const float4*>(x + c * kChunk + 4);
  };
  load_weights(warp);
  if (!waited)
    pdl_wait();
  waited = true;
  load_activations(warp);
#pragma unroll 1
  for (int base = 0; base < chunks; base += kRoundChunks) {
    const int here = min(kRoundChunks, chunks - base);
#pragma unroll 1
    for (int c = warp; c < here; c += kInnerWarps) {
      Raw<W, 8> raw[kFewTiles][2];
#pragma unroll
      for (int i = 0; i < kFewTiles; ++i)
        raw[i][0] = next[i][0], raw[i][1] = next[i][1];
      float4 v0 = x0, v1 = x1;
      load_weights(base + c + kInnerWarps);
      load_activations(base + c + kInnerWarps);
      float2 back = make_float2(1.f, 1.f);
      if (kHalf) {
        float most = fmaxf(fmaxf(fmaxf(fabsf(v0.x), fabsf(v0.y)), fmaxf(fabsf(v0.z), fabsf(v0.w))), fmaxf(fmaxf(fabsf(v1.x), fabsf(v1.y)), fmaxf(fabsf(v1.z), fabsf(v1.w))));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        float to, unit;
        range_of(most, to, unit);
        v0.x *= to, v0.y *= to, v0.z *= to, v0.w *= to, v1.x *= to, v1.y *= to, v1.z *= to, v1.w *= to;
        back = make_float2(__shfl_sync(0xffffffffu, unit, 8 * t), __shfl_sync(0xffffffffu, unit, 8 * t + 4));  // of rows 2 t and 2 t + 1
      }
      uint2 column[2][kPieces];
      cut_four<W>(v0, column[0]), cut_four<W>(v1, column[1]);
#pragma unroll
      for (int i = 0; i < kFewTiles; ++i) {
        uint32_t up[kWeightPieces][4], low[kWeightPieces][4];
        pieces_of<W, 8>(raw[i][0], up), pieces_of<W, 8>(raw[i][1], low);
        float d[kPieces][4] = {};
#pragma unroll
        for (int s = 0; s < 2; ++s)
          add_product<W, 4>(d, up, low, 2 * s, column[s]);
        float* to = &sh.parts[c][2 * t][16 * i + g];
        to[0] = total(d, 0) * back.x, to[kFewTiles * 16] = total(d, 1) * back.y, to[8] = total(d, 2) * back.x, to[kFewTiles * 16 + 8] = total(d, 3) * back.y;
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const int at = tid + i * kThreads, row = at / (kFewTiles * 16), r = at % (kFewTiles * 16);
      if (row < rows && r < 16 * tiles) {
        float term[kRoundChunks];
#pragma unroll
        for (int c = 0; c < kRoundChunks; ++c)
          term[c] = c < here ? sh.parts[c][row][r] : 0.f;
#pragma unroll
        for (int c = 0; c < kRoundChunks; ++c)
          sum[i] += term[c];
      }
    }
    __syncthreads();  // the parts may be written again
  }
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    const int at = tid + i * kThreads;
    sh.result[at / (kFewTiles * 16)][at % (kFewTiles * 16)] = sum[i];
  }
}

template <class W, int BLOCK, bool VEC>
__device__ __forceinline__ void inner_many(const AdapterParams& p, ManyShared<W>& sh, const int (&ranks)[kAdapterMaxMatrices], int adapter, const int* rowsOf, int rows, int firstTile,
                                           int tiles, int part, int chunks, bool& waited) {
  constexpr int kInnerWarps = inner_warps(BLOCK), kThreads = kInnerWarps * kWarp, kPieces = Format<W>::kPieces, kWeightPieces = Format<W>::kWeightPieces, kRowsEach = 32 / kInnerWarps;
  constexpr int kAhead = ManyShared<W>::kAhead;
  constexpr bool kHalf = Format<W>::kHalf;
  const int tid = threadIdx.x, warp = tid / kWarp, lane = tid % kWarp, g = lane >> 2, t = lane & 3;
  const int64_t from = int64_t(part) * chunks * kChunk;
  const int length = chunks * kChunk, spans = (length + kSpan - 1) / kSpan;
  // ---- weights: pieces of 16 bytes, those of a span in a row; zeros past the end of the part
  constexpr int kPiece = 16 / int(sizeof(W)), kAcross = kSpan / kPiece, kRanksEach = kManyTiles * 16 * kAcross / kThreads;
  const W* source[kRanksEach];
#pragma unroll
  for (int i = 0; i < kRanksEach; ++i) {
    const int r = tid / kAcross + i * (kThreads / kAcross);
    const Tile<W> tile = tile_of<W>(p, ranks, adapter, firstTile + min(r / 16, tiles - 1));
    source[i] = tile.a + from + min(tile.first + r % 16, tile.rank - 1) * p.k + tid % kAcross * kPiece;
  }
  auto fetch_weights = [&](int span) {
    const int at = span * kSpan + tid % kAcross * kPiece;
#pragma unroll
    for (int i = 0; i < kRanksEach; ++i) {
      const int r = tid / kAcross + i * (kThreads / kAcross);
      if (span < spans && r < 16 * tiles) {
        uint8_t* to = sh.weights[span % (kAhead + 1)] + r * ManyShared<W>::kWeightPitch + tid % kAcross * 16;
        if constexpr (VEC) {
          const uint32_t bytes = at < length ? 16u : 0u;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to)), "l"(source[i] + (bytes ? span * kSpan : 0)), "r"(bytes) : "memory");
        } else {
          for (int e = 0; e < kPiece; ++e)
            reinterpret_cast<W*>(to)[e] = at < length ? source[i][span * kSpan + e] : W(0.f);
        }
      }
    }
  };
  auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
  // ---- activations: a warp has two rows, a lane four activations of each, which it brings and cuts itself; zeros past the last row and the end of the part
  const float* activations[kRowsEach];
#pragma unroll
  for (int i = 0; i < kRowsEach; ++i)
    activations[i] = p.x + int64_t(rowsOf[min(warp + kInnerWarps * i, rows - 1)]) * p.k + from;
  auto fetch_activations = [&](int span) {
    const int at = span * kSpan + 4 * lane;
#pragma unroll
    for (int i = 0; i < kRowsEach; ++i) {
      const int row = warp + kInnerWarps * i;
      const uint32_t bytes = row < rows && at < length ? 16u : 0u;
      if (span < spans)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(&sh.uncut[span % kAhead][row][4 * lane])), "l"(activations[i] + (bytes ? at : 0)), "r"(bytes) : "memory");
    }
  };
  auto stage = [&](int span) {
    const int buffer = span & 1;
#pragma unroll
    for (int i = 0; i < kRowsEach; ++i) {
      const int row = warp + kInnerWarps * i;
      float4 v = *reinterpret_cast<const float4*>(&sh.uncut[span % kAhead][row][4 * lane]);
      if (kHalf) {
        float most = fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w)));
#pragma unroll
        for (int o = 1; o < kChunk / 4; o <<= 1)
          most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        float to, back;
        range_of(most, to, back);
        v.x *= to, v.y *= to, v.z *= to, v.w *= to;
        if (lane % (kChunk / 4) == 0)
          sh.back[buffer][lane / (kChunk / 4)][row] = back;
      }
      uint2 piece[kPieces];
      cut_four<W>(v, piece);
#pragma unroll
      for (int q = 0; q < kPieces; ++q)
        *reinterpret_cast<uint2*>(&sh.x[buffer][q][row][4 * lane]) = piece[q];
    }
  };
#pragma unroll
  for (int span = 0; span < kAhead; ++span)
    fetch_weights(span);
  if (!waited)
    pdl_wait();
  waited = true;
#pragma unroll
  for (int span = 0; span < kAhead; ++span) {
    fetch_activations(span);
    commit();
  }
  asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
  stage(0);
  // ---- products: a warp has a tile, and COUNT eights of rows from `begin` on
  const int across = tiles > 4 ? 8 : 4, own = min(warp % across, tiles - 1), begin = warp / across * (tiles > 4 ? 2 : 1);
  static_assert(kInnerWarps == 16 && kManyTiles == 8, "a warp for each tile and half or quarter of the rows");
  auto run = [&](auto count) {
    constexpr int kCount = decltype(count)::value;
    float acc[kCount][4] = {};
#pragma unroll 1
    for (int span = 0; span < spans; ++span) {
      const int buffer = span & 1;
      __syncthreads();  // this span is there, and everybody is done with the one before
      fetch_weights(span + kAhead);
      fetch_activations(span + kAhead);
      commit();
      const uint8_t* const weights = sh.weights[span % (kAhead + 1)] + own * 16 * ManyShared<W>::kWeightPitch;
#pragma unroll
      for (int c = 0; c < kSpan / kChunk; ++c) {
        uint32_t w[2][kWeightPieces][4];  // of both halves of the chunk
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          if constexpr (sizeof(W) == 2) {
            ldmatrix4(w[s][0], weights + (lane & 15) * ManyShared<W>::kWeightPitch + (c * kChunk + s * 16 + (lane >> 4) * 8) * 2);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float2 pair = *reinterpret_cast<const float2*>(weights + (8 * (e & 1) + g) * ManyShared<W>::kWeightPitch + (c * kChunk + s * 16 + (e >> 1) * 8 + 2 * t) * 4);
#pragma unroll
              for (int q = 0; q < kWeightPieces; ++q)
                w[s][q][e] = cut_pair(pair.x, pair.y);
            }
          }
        }
#pragma unroll
        for (int j = 0; j < kCount; ++j) {
          uint32_t column[kPieces][4];
#pragma unroll
          for (int q = 0; q < kPieces; ++q)
            ldmatrix4(column[q], &sh.x[buffer][q][8 * (begin + j) + (lane & 7)][c * kChunk + (lane >> 3) * 8]);
          float d[kPieces][4] = {};
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int q = kWeightPieces - 1; q >= 0; --q)
#pragma unroll
              for (int order = kPieces - 1; order >= 0; --order)
                if (order - q >= 0)
                  mma<kHalf>(d[order], w[s][q][0], w[s][q][1], w[s][q][2], w[s][q][3], column[order - q][2 * s], column[order - q][2 * s + 1]);
          float2 back = make_float2(1.f, 1.f);
          if (kHalf)
            back = *reinterpret_cast<const float2*>(&sh.back[buffer][c][8 * (begin + j) + 2 * t]);
          acc[j][0] += total(d, 0) * back.x, acc[j][1] += total(d, 1) * back.y, acc[j][2] += total(d, 2) * back.x, acc[j][3] += total(d, 3) * back.y;
        }
      }
      asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");  // the next span's
      if (span + 1 < spans)
        stage(span + 1);
    }
    __syncthreads();  // the weights are done with: their place takes the results
    if (warp % across >= tiles)
      return;
#pragma unroll
    for (int j = 0; j < kCount; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        sh.result[8 * (begin + j) + 2 * t + (e & 1)][16 * own + g + 8 * (e >> 1)] = acc[j][e];
  };
  if (tiles > 4)
    run(std::integral_constant<int, 2>());
  else
    run(std::integral_constant<int, 1>());
}

template <class W, bool PAIR, int BLOCK>
__global__ void __launch_bounds__(inner_warps(BLOCK) * kWarp, BLOCK > 1 ? 1 : 2) inner_products_kernel(const __grid_constant__ AdapterParams p) {
  extern __shared__ __align__(16) uint8_t innerRaw[];
  InnerShared& sh = *reinterpret_cast<InnerShared*>(innerRaw);  // its results are where ManyShared has them
  constexpr int kThreads = inner_warps(BLOCK) * kWarp;
  __shared__ int rowsOf[inner_warps(BLOCK)][32];
  pdl_launch_dependents();
  const int tid = threadIdx.x, warp = tid / kWarp;
  const int chunks = int(p.k) / kChunk / kParts, part = blockIdx.x, lane = tid % kWarp;
  // Items of a lane's adapter. By eights of rows (kFew) where all of them run at once, one CTA an SM: 40 rows of two tiles of ranks, k = 12288; where they come one after the
  // other, 128 rows of three tiles took 14.1 us in all instead of 13.1 from staged weights. Of those, half the tiles an item (kHalf) where these run at once: a pair of rank 64 for
  // 128 rows 23.5 us instead of 25.2. Rows of an adapter that has no more than eight always go the first way, so that their results do not depend on what else there is.
  enum { kFew, kHalf, kAll, kWays };
  auto tiles_of = [](const Block& block) {
    int tiles = 0;
#pragma unroll
    for (int i = 0; i < kAdapterMaxMatrices; ++i)
      tiles += (block.rank[i] + 15) / 16;
    return tiles;
  };
  auto items_of = [&](const Block& block, int way) {
    const int members = __popc(block.group), tiles = tiles_of(block), each = way == kHalf ? kManyTiles / 2 : kManyTiles;
    return way == kFew || members <= 8 ? (tiles + kFewTiles - 1) / kFewTiles * ((members + 7) / 8) : (tiles + each - 1) / each;
  };
  // The items of all blocks are counted through, so that the first CTAs have one each. (By a grid of blocks and items, the second items of a block of 512 rows started when
  // the first ones were done, behind CTAs that had none: 39.0 us instead of 35.3. 128 rows of three projections took 13.2 us instead of 13.5.)
  const int slots = int(gridDim.y * gridDim.z);
  int way = kFew, blocksUpTo = 0, all = 0;
  Block block;
  if constexpr (BLOCK == 1) {
    block = find_block<8, PAIR>(p, 0, blockIdx.x == 0 && blockIdx.z == 0 && warp == 0);
    blocksUpTo = all = __reduce_add_sync(0xffffffffu, items_of(block, kFew));
  } else {
    constexpr int kBlocks = kAdapterSlabRows / 32;
    __shared__ int items[kWays][kBlocks];
    const int blocks = int(gridDim.y);
    for (int b = warp; b < blocks; b += inner_warps(BLOCK)) {
      const Block other = find_block<8 * BLOCK, PAIR>(p, b, blockIdx.x + blockIdx.y + blockIdx.z == 0);
#pragma unroll
      for (int i = 0; i < kWays; ++i) {
        const int sum = __reduce_add_sync(0xffffffffu, items_of(other, i));
        if (lane == 0)
          items[i][b] = sum;
      }
    }
    __syncthreads();
    int here[kWays], total[kWays];
#pragma unroll
    for (int i = 0; i < kWays; ++i)
      here[i] = lane < blocks ? items[i][lane] : 0, total[i] = __reduce_add_sync(0xffffffffu, here[i]);
    way = total[kFew] <= slots / 2 ? kFew : total[kHalf] <= slots / 2 ? kHalf : kAll;
    blocksUpTo = running_sum(way == kFew ? here[kFew] : way == kHalf ? here[kHalf] : here[kAll]);
    all = way == kFew ? total[kFew] : way == kHalf ? total[kHalf] : total[kAll];
  }
  bool waited = false;
#pragma unroll 1
  for (int slot = blockIdx.y + gridDim.y * blockIdx.z; slot < all; slot += slots) {
    int index = slot;
    if constexpr (BLOCK > 1) {
      const int which = __ffs(__ballot_sync(0xffffffffu, blocksUpTo > slot)) - 1;
      if (which)
        index -= __shfl_sync(0xffffffffu, blocksUpTo, which - 1);
      block = find_block<8 * BLOCK, PAIR>(p, which, false);
    }
    const int tilesOwn = tiles_of(block), own = items_of(block, way), upTo = running_sum(own);
    const int holder = __ffs(__ballot_sync(0xffffffffu, upTo > index)) - 1;
    const int within = index - __shfl_sync(0xffffffffu, upTo - own, holder), adapter = __shfl_sync(0xffffffffu, block.which, holder);
    const int tilesAll = __shfl_sync(0xffffffffu, tilesOwn, holder);
    const uint32_t group = __shfl_sync(0xffffffffu, block.group, holder);
    int ranks[kAdapterMaxMatrices];
#pragma unroll
    for (int i = 0; i < kAdapterMaxMatrices; ++i)
      ranks[i] = __shfl_sync(0xffffffffu, block.rank[i], holder);
    __syncthreads();  // the rows and the sums of the item before are done with
    list_rows(rowsOf[warp], group, block.base);
    __syncwarp();
    int rows = __popc(group), first, tiles;
    uint64_t addresses = 0;
    for (int i = 0; i < (PAIR ? 2 : p.count); ++i)
      addresses |= p.adapters[i][adapter].a;
    const bool aligned = addresses % 16 == 0;
    const int* list = rowsOf[warp];
    if (BLOCK == 1 || way == kFew || rows <= 8) {
      const int batches = (tilesAll + kFewTiles - 1) / kFewTiles, row0 = within / batches * 8;
      first = within % batches * kFewTiles, tiles = min(kFewTiles, tilesAll - first), list += row0, rows = min(8, rows - row0);
      if (aligned)
        inner_few<W, BLOCK, true>(p, sh, ranks, adapter, list, rows, first, tiles, part, chunks, waited);
      else
        inner_few<W, BLOCK, false>(p, sh, ranks, adapter, list, rows, first, tiles, part, chunks, waited);
    } else if constexpr (BLOCK > 1) {
      const int each = way == kHalf ? kManyTiles / 2 : kManyTiles;
      first = within * each, tiles = min(each, tilesAll - first);
      if (aligned)
        inner_many<W, BLOCK, true>(p, *reinterpret_cast<ManyShared<W>*>(innerRaw), ranks, adapter, list, rows, first, tiles, part, chunks, waited);
      else
        inner_many<W, BLOCK, false>(p, *reinterpret_cast<ManyShared<W>*>(innerRaw), ranks, adapter, list, rows, first, tiles, part, chunks, waited);
    }
    __syncthreads();
    constexpr int kMost = kManyTiles * 16;
    const int r = tid % kMost;
    if (r < tiles * 16) {
      const Tile<W> tile = tile_of<W>(p, ranks, adapter, first + r / 16);
      if (tile.first + r % 16 < tile.rank)
        for (int row = tid / kMost; row < rows; row += kThreads / kMost)
          p.inner[inner_at<BLOCK>(part, list[row], tile.matrix, tile.first + r % 16)] = sh.result[row][r];
    }
  }
  if (!waited)
    pdl_wait();  // the end of this kernel means the end of all before it
}

// ---- outer products: grid (CTAs of a block, blocks) ----
// A CTA has some units of columns of one adapter and matrix, or of several, dealt to its warps in turn. A warp brings its units' weights through two stages of shared
// memory of its own, up to 128 bytes of a column at a time, while it multiplies the stage before: nobody waits for anybody. (Weights straight from global memory to where an MMA
// wants them are eight pieces of 32 bytes in eight lines a load: 512 rows of rank 64 to 12288 columns took 49 us.)
constexpr int kStageBytes = 128, kStagePitch = kStageBytes + 16;  // 16 bytes more: eight columns in eight different groups of banks
template <class W> constexpr int stage_ranks() { return kStageBytes / int(sizeof(W)); }

template <class W> struct OuterShared {
  __align__(16) uint8_t weights[kOuterWarps][2][kUnit * kStagePitch];
  __align__(16) uint32_t inner[Format<W>::kPieces][kInner / 2];  // inner products, scaled and cut: [piece][tile of 16 ranks][row][pair of ranks], pairs in the order 0 4 1 5 2 6 3 7
  __align__(16) float uncut[Format<W>::kHalf ? kInner : 4];      // fp16: before they are cut
  uint32_t largest[2][32];                                       // fp16: of a row of them and a matrix of a pair, the bits of its magnitude
  __align__(8) float back[2][32];                                // fp16: what brings their products back to scale
  int rows[32];
};
static_assert(2 * kAdapterMaxRank * 8 <= kInner, "eight rows of a pair of the largest ranks fit");
static_assert(sizeof(OuterShared<__half>) <= 113 * 1024 && sizeof(OuterShared<float>) <= 113 * 1024, "two CTAs an SM");

// A warp's weights of one matrix.
template <class W> struct Weights {
  const W* b;
  int rank, steps;  // a step is a stage
  bool whole;       // whole pieces of 16 bytes
};
template <class W> __device__ __forceinline__ Weights<W> weights_of(const infdev_adapter* records, int adapter, int rank, float& scale) {
  Weights<W> w{nullptr, rank, (rank + stage_ranks<W>() - 1) / stage_ranks<W>(), false};
  if (rank) {
    w.b = reinterpret_cast<const W*>(records[adapter].b), scale = records[adapter].scale;
    w.whole = (rank * int(sizeof(W))) % 16 == 0 && (reinterpret_cast<uintptr_t>(w.b) & 15) == 0;
  }
  return w;
}

// Ranks firstRank .. of a unit's columns into a stage, zeros past the last rank; columns past the last of the matrix are repeated. Column 2 g + h becomes row 8 h + g, so that a lane
// ends up with two consecutive columns.
template <class W> __device__ __forceinline__ void stage_weights(uint8_t* stage, const Weights<W>& w, int firstRank, int column, int n) {
  constexpr int kPiece = 16 / int(sizeof(W));
  const int count = min(stage_ranks<W>(), (w.rank - firstRank + 15) / 16 * 16) / kPiece;  // pieces of 16 bytes a column, in whole tiles of ranks
  const int lane = threadIdx.x % kWarp, piece = lane % 8, h = lane / 8, r = firstRank + piece * kPiece;
  if (piece >= count)
    return;
  uint8_t* const to = stage + ((h & 1) * 8 + (h >> 1)) * kStagePitch + piece * 16;  // of the first four columns; the next four are two rows on
  if (w.whole) {
    const uint32_t shared = smem_u32(to), bytes = r < w.rank ? 16u : 0u;
    auto copy = [&](int i, const W* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(shared + 2 * i * kStagePitch), "l"(from), "r"(bytes) : "memory"); };
    const W* from = w.b + ((column + h) * w.rank + min(r, w.rank - kPiece));  // fits 32 bits: 2^20 columns of 256 ranks
    if (column + kUnit <= n) {
#pragma unroll
      for (int i = 0; i < kUnit / 4; ++i, from += 4 * w.rank)  // four columns at a time: 4 i + h
        copy(i, from);
    } else {
#pragma unroll 1
      for (int i = 0; i < kUnit / 4; ++i)
        copy(i, from + (min(column + 4 * i + h, n - 1) - column - h) * w.rank);
    }
    return;
  }
#pragma unroll 1
  for (int i = 0; i < kUnit / 4; ++i) {
    const W* const from = w.b + (min(column + 4 * i + h, n - 1) * w.rank + r);
#pragma unroll
    for (int e = 0; e < kPiece; ++e)
      reinterpret_cast<W*>(to + 2 * i * kStagePitch)[e] = r + e < w.rank ? from[e] : W(0.f);
  }
}

// d: columns 2 g and 2 g + 1 of rows 2 t and 2 t + 1 of every eight, plus the products of TILES tiles of ranks of a stage. `unit`, `inner`: from the first of them on.
template <class W, int NT, int TILES> __device__ __forceinline__ void multiply_tiles(float (&d)[NT][4], const uint8_t* unit, const uint32_t* inner) {
  constexpr int kPieces = Format<W>::kPieces, kWeightPieces = Format<W>::kWeightPieces, kRows = 8 * NT;
  const int lane = threadIdx.x % kWarp, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int tile = 0; tile < TILES; ++tile) {
    uint32_t w[kWeightPieces][4];  // upper, lower half, then of the next eight ranks
    if constexpr (sizeof(W) == 2) {
      ldmatrix4(w[0], unit + (lane & 15) * kStagePitch + tile * 32 + (lane >> 4) * 16);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float2 v = *reinterpret_cast<const float2*>(unit + (8 * (e & 1) + g) * kStagePitch + tile * 64 + (e >> 1) * 32 + t * 8);
#pragma unroll
        for (int q = 0; q < kWeightPieces; ++q)
          w[q][e] = cut_pair(v.x, v.y);
      }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      uint2 column[kPieces];
#pragma unroll
      for (int q = 0; q < kPieces; ++q)
        column[q] = *reinterpret_cast<const uint2*>(inner + q * (kInner / 2) + (tile * kRows + 8 * j + g) * 8 + 2 * t);
#pragma unroll
      for (int order = kPieces - 1; order >= 0; --order)
#pragma unroll
        for (int q = kWeightPieces - 1; q >= 0; --q)
          if (order - q >= 0)
            mma<Format<W>::kHalf>(d[j], w[q][0], w[q][1], w[q][2], w[q][3], column[order - q].x, column[order - q].y);
    }
  }
}
template <class W, int NT> __device__ __forceinline__ void multiply(float (&d)[NT][4], const OuterShared<W>& sh, const uint8_t* unit, int tiles, int firstTile) {
  constexpr int kTileBytes = 16 * sizeof(W), kMost = stage_ranks<W>() / 16;
  const uint32_t* inner = &sh.inner[0][firstTile * 8 * NT * 8];
  if (tiles == kMost) {  // without a branch between them, a tile's operands are on their way while the one before is multiplied
    multiply_tiles<W, NT, kMost>(d, unit, inner);
    return;
  }
#pragma unroll 1
  for (int tile = 0; tile < tiles; ++tile)
    multiply_tiles<W, NT, 1>(d, unit + tile * kTileBytes, inner + tile * 8 * NT * 8);
}

// Two columns of a row, or the one that exists. VEC: they are two, on an 8-byte boundary.
template <bool VEC> __device__ __forceinline__ float2 load_columns(const float* from, int left) {
  if constexpr (VEC)
    return *reinterpret_cast<const float2*>(from);
  return make_float2(from[0], left > 1 ? from[1] : 0.f);
}
template <bool VEC> __device__ __forceinline__ void store_columns(float* to, const float2& v, int left) {
  if constexpr (VEC) {
    *reinterpret_cast<float2*>(to) = v;
    return;
  }
  to[0] = v.x;
  if (left > 1)
    to[1] = v.y;
}

// Units `first` .. `last` - 1 of a matrix (of both, of a pair) for up to 8 NT rows of an adapter. BLOCK: of the launch, in eights of rows.
template <class W, bool PAIR, int NT, int BLOCK, bool VEC>
__device__ __forceinline__ void run_units(const AdapterParams& p, OuterShared<W>& sh, int matrix, int adapter, int rank0, int rank1, int row0, int rowCount, int first, int last, bool& waited) {
  constexpr int kRows = 8 * NT, kPieces = Format<W>::kPieces, kThreads = kOuterWarps * kWarp, kRanks = stage_ranks<W>(), kHalves = PAIR ? 2 : 1;
  constexpr bool kHalf = Format<W>::kHalf;
  const int tid = threadIdx.x, warp = tid / kWarp, lane = tid % kWarp, g = lane >> 2, t = lane & 3;
  const int live = min(kRows, rowCount - row0), n = int(p.n[matrix]);
  const int tiles0 = (rank0 + 15) / 16, tiles1 = (rank1 + 15) / 16, tiles = tiles0 + tiles1;
  float scale0 = 0.f, scale1 = 0.f;
  const Weights<W> w0 = weights_of<W>(p.adapters[matrix], adapter, rank0, scale0), w1 = weights_of<W>(PAIR ? p.adapters[1] : nullptr, adapter, PAIR ? rank1 : 0, scale1);
  const int steps = w0.steps + w1.steps;
  auto fetch = [&](int unit, int step, int stage) {
    if (unit < last) {
      if (PAIR && step >= w0.steps)
        stage_weights(sh.weights[warp][stage], w1, (step - w0.steps) * kRanks, unit * kUnit, n);
      else
        stage_weights(sh.weights[warp][stage], w0, step * kRanks, unit * kUnit, n);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (steps)
    fetch(first + warp, 0, 0);  // on its way while the inner products are waited for
  if (!waited)
    pdl_wait();
  waited = true;
  // ---- what is added to: lane (g, t) has columns 2 g and 2 g + 1 of a unit and rows 2 t, 2 t + 1 of every eight
  const float* const before[2] = {p.residual[matrix], p.residual[matrix + (PAIR ? 1 : 0)]};
  float* const y = p.y[matrix];
  int rowAt[NT][2];  // fits 32 bits: 512 rows of 2^20 columns. Rows past the last are repeated, and not stored.
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 2; ++e)
      rowAt[j][e] = sh.rows[min(row0 + 8 * j + 2 * t + e, rowCount - 1)] * n;
  auto load_rows = [&](float2 (&to)[kHalves][2], int unit, int j) {
    const int column = min(unit * kUnit + 2 * g, (n - 1) / 2 * 2);  // columns past the last too
#pragma unroll
    for (int half = 0; half < kHalves; ++half)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        to[half][e] = load_columns<VEC>(before[half] + (rowAt[j][e] + column), n - column);
  };
  // Few rows are on their way one unit ahead, many while their unit's products are taken: a unit ahead, four projections of 512 rows took 42.4 instead of 37.2 us.
  constexpr bool kAhead = NT == 1;
  float2 held[NT][kHalves][2], coming[kHalves][2];
  if (kAhead && first + warp < last)
    load_rows(coming, first + warp, 0);
  // ---- the inner products: the sum of their parts, scaled and cut
  const int values = tiles * kRows * 16;
  if (kHalf) {
    if (tid < kHalves * kRows)
      sh.largest[tid / kRows][tid % kRows] = 0;
    __syncthreads();
  }
  auto cut = [&](int i, float4 v) {
    uint2 piece[kPieces];
    cut_four<W>(v, piece);
    const int pair = i % 16 / 2, at = i / 16 * 8 + pair % 4 * 2 + pair / 4;
#pragma unroll
    for (int q = 0; q < kPieces; ++q)
      sh.inner[q][at] = piece[q].x, sh.inner[q][at + 2] = piece[q].y;
  };
  constexpr int kTogether = NT > 1 ? 2 : 1;  // of four ranks of a row, their parts on their way together
#pragma unroll 1
  for (int base = tid * 4; base < values; base += kTogether * kThreads * 4) {
    float4 part[kTogether][kParts];
    int left[kTogether];
    float scale[kTogether];
#pragma unroll
    for (int k = 0; k < kTogether; ++k) {
      const int i = min(base + k * kThreads * 4, values - 4), tile = i / (kRows * 16), row = i / 16 % kRows;
      const bool second = PAIR && tile >= tiles0;
      const int r = (tile - (second ? tiles0 : 0)) * 16 + i % 16;
      left[k] = row < live ? (second ? rank1 : rank0) - r : 0, scale[k] = second ? scale1 : scale0;
      // rows and ranks past the last are taken from others, and not used
      const float* from = p.inner + inner_at<BLOCK>(0, sh.rows[min(row0 + row, rowCount - 1)], matrix + (second ? 1 : 0), r);
      const size_t step = inner_at<BLOCK>(1, 0, 0, 0);
#pragma unroll
      for (int e = 0; e < kParts; ++e)
        part[k][e] = __ldcg(reinterpret_cast<const float4*>(from + e * step));
    }
#pragma unroll
    for (int k = 0; k < kTogether; ++k) {
      const int i = base + k * kThreads * 4;
      if (i >= values)
        break;
      float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int e = 0; e < kParts; ++e)
        v[0] += part[k][e].x, v[1] += part[k][e].y, v[2] += part[k][e].z, v[3] += part[k][e].w;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        v[e] = e < left[k] ? v[e] * scale[k] : 0.f;
      if constexpr (kHalf) {
        *reinterpret_cast<float4*>(sh.uncut + i) = make_float4(v[0], v[1], v[2], v[3]);
        atomicMax(&sh.largest[PAIR && i >= tiles0 * kRows * 16][i / 16 % kRows], __float_as_uint(fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])))));
      } else {
        cut(i, make_float4(v[0], v[1], v[2], v[3]));
      }
    }
  }
  if constexpr (kHalf) {
    __syncthreads();
    if (tid < kHalves * kRows) {
      float to;
      range_of(__uint_as_float(sh.largest[tid / kRows][tid % kRows]), to, sh.back[tid / kRows][tid % kRows]);
    }
#pragma unroll 1
    for (int i = tid * 4; i < values; i += kThreads * 4) {
      float to, back;
      range_of(__uint_as_float(sh.largest[PAIR && i >= tiles0 * kRows * 16][i / 16 % kRows]), to, back);
      const float4 v = *reinterpret_cast<const float4*>(sh.uncut + i);
      cut(i, make_float4(v.x * to, v.y * to, v.z * to, v.w * to));
    }
  }
  __syncthreads();  // the inner products are there
  // ---- columns
  int stage = 0;
#pragma unroll 1
  for (int unit = first + warp; unit < last; unit += kOuterWarps) {
    if (kAhead) {
#pragma unroll
      for (int half = 0; half < kHalves; ++half)
        held[0][half][0] = coming[half][0], held[0][half][1] = coming[half][1];
      load_rows(coming, min(unit + kOuterWarps, last - 1), 0);
    } else {
#pragma unroll
      for (int j = 0; j < NT; ++j)
        load_rows(held[j], unit, j);
    }
    float d[kHalves][NT][4];
#pragma unroll
    for (int i = 0; i < kHalves * NT * 4; ++i)
      d[i / (4 * NT)][i / 4 % NT][i % 4] = 0.f;
#pragma unroll
    for (int half = 0; half < kHalves; ++half) {
#pragma unroll 1
      for (int step = half ? w0.steps : 0; step < (half ? steps : w0.steps); ++step, stage ^= 1) {
        fetch(step + 1 < steps ? unit : unit + kOuterWarps, step + 1 < steps ? step + 1 : 0, stage ^ 1);
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncwarp();
        const int firstRank = (step - (half ? w0.steps : 0)) * kRanks, rank = half ? rank1 : rank0;
        multiply<W, NT>(d[half], sh, sh.weights[warp][stage], min(kRanks, rank - firstRank + 15) / 16, (half ? tiles0 : 0) + firstRank / 16);
        __syncwarp();  // the stage may be filled again
      }
    }
    const int column = unit * kUnit + 2 * g;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      if (8 * j >= live)
        break;
      const float2(&rows)[kHalves][2] = held[j];
      float2 back[kHalves];  // of both rows
#pragma unroll
      for (int half = 0; half < kHalves; ++half)
        back[half] = kHalf ? *reinterpret_cast<const float2*>(&sh.back[half][8 * j + 2 * t]) : make_float2(1.f, 1.f);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (8 * j + e >= live)
          break;
        const float unitOf = e ? back[0].y : back[0].x;
        float2 v = rows[0][e];
        v.x += d[0][j][e] * unitOf, v.y += d[0][j][2 + e] * unitOf;
        if constexpr (PAIR) {
          const float2 u = rows[1][e];
          const float upOf = e ? back[1].y : back[1].x;
          v.x = silu_f(v.x) * (u.x + d[1][j][e] * upOf), v.y = silu_f(v.y) * (u.y + d[1][j][2 + e] * upOf);
        }
        if (8 * j + 2 * t + e < live && column < n)
          store_columns<VEC>(y + (rowAt[j][e] + column), v, n - column);
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();  // the inner products are done with
}

template <class W, bool PAIR, int NT>
__global__ void __launch_bounds__(kOuterWarps* kWarp, 2) outer_products_kernel(const __grid_constant__ AdapterParams p) {
  extern __shared__ __align__(16) uint8_t outerRaw[];
  OuterShared<W>& sh = *reinterpret_cast<OuterShared<W>*>(outerRaw);
  pdl_launch_dependents();
  const int tid = threadIdx.x, warp = tid / kWarp;
  const Block block = find_block<8 * NT, PAIR>(p, blockIdx.y, false);
  // What a unit of columns costs, in hundreds of cycles or so: itself, the rows that it reads and writes, and the weights, which are multiplied with eight rows at a time. Rows that are
  // added to in place and have nothing to add are left alone.
  const int matrices = PAIR ? 1 : p.count;
  const int eights = (__popc(block.group) + 7) / 8;
  int weight[kAdapterMaxMatrices], units[kAdapterMaxMatrices], own = 0;
#pragma unroll
  for (int i = 0; i < kAdapterMaxMatrices; ++i) {
    weight[i] = units[i] = 0;
    if (i < matrices) {
      units[i] = (int(p.n[i]) + kUnit - 1) / kUnit;
      const int tiles = (block.rank[i] + 15) / 16 + (PAIR ? (block.rank[1] + 15) / 16 : 0);
      if (block.leads && (tiles || PAIR || p.residual[i] != p.y[i]))
        weight[i] = 16 + eights * (PAIR ? 10 : 5) + tiles * (1 + eights);
      own += units[i] * weight[i];
    }
  }
  const int upTo = running_sum(own), total = __shfl_sync(0xffffffffu, upTo, 31), share = (total + int(gridDim.x) - 1) / int(gridDim.x);
  const int end = min(total, share * (int(blockIdx.x) + 1));
  bool waited = false;
#pragma unroll 1
  for (int at = share * int(blockIdx.x); at < end;) {
    // the adapter and the matrix that `at` falls into, and the units whose first cost lies in at .. end - 1
    const int holder = __ffs(__ballot_sync(0xffffffffu, upTo > at)) - 1;
    int from = __shfl_sync(0xffffffffu, upTo - own, holder), matrix = 0, each = 0, count = 0, rank0 = 0;
    for (;; ++matrix) {
      each = __shfl_sync(0xffffffffu, matrix == 0 ? weight[0] : matrix == 1 ? weight[1] : matrix == 2 ? weight[2] : weight[3], holder);
      rank0 = __shfl_sync(0xffffffffu, matrix == 0 ? block.rank[0] : matrix == 1 ? block.rank[1] : matrix == 2 ? block.rank[2] : block.rank[3], holder);
      count = matrix == 0 ? units[0] : matrix == 1 ? units[1] : matrix == 2 ? units[2] : units[3];
      if (at < from + each * count)
        break;
      from += each * count;
    }
    const int rank1 = PAIR ? __shfl_sync(0xffffffffu, block.rank[1], holder) : 0;
    const int first = (at - from + each - 1) / each, last = min(count, (end - from + each - 1) / each);
    const uint32_t group = __shfl_sync(0xffffffffu, block.group, holder);
    const int adapter = __shfl_sync(0xffffffffu, block.which, holder), rowCount = __popc(group);
    if (first < last) {
      if (warp == 0)
        list_rows(sh.rows, group, block.base);
      __syncthreads();
      const uintptr_t addresses = reinterpret_cast<uintptr_t>(p.y[matrix]) | reinterpret_cast<uintptr_t>(p.residual[matrix]) | reinterpret_cast<uintptr_t>(p.residual[matrix + (PAIR ? 1 : 0)]);
      const bool vec = p.n[matrix] % 2 == 0 && addresses % 8 == 0;
      const bool many = NT > 1 && rowCount > 8 && ((rank0 + 15) / 16 + (rank1 + 15) / 16) * 16 * 8 * NT <= kInner;
#pragma unroll 1
      for (int row0 = 0; row0 < rowCount;) {
        auto run = [&](auto eights, auto aligned) {
          run_units<W, PAIR, decltype(eights)::value, NT, decltype(aligned)::value>(p, sh, matrix, adapter, rank0, rank1, row0, rowCount, first, last, waited);
          row0 += 8 * decltype(eights)::value;
        };
        using One = std::integral_constant<int, 1>;
        using Many = std::integral_constant<int, NT>;
        if (many)
          vec ? run(Many(), std::true_type()) : run(Many(), std::false_type());
        else
          vec ? run(One(), std::true_type()) : run(One(), std::false_type());
      }
    }
    at = from + each * count;
  }
  if (!waited)
    pdl_wait();
}

template <class W, bool PAIR, int NT> cudaError_t launch_blocks(const AdapterParams& p, int sms, cudaStream_t stream) {
  constexpr int kRows = 8 * NT;
  constexpr size_t kInnerBytes = NT > 1 ? sizeof(ManyShared<W>) : sizeof(InnerShared);
  const auto inner = inner_products_kernel<W, PAIR, NT>;
  const auto outer = outer_products_kernel<W, PAIR, NT>;
  static PerDeviceOnce innerConfigured, outerConfigured;
  if (const cudaError_t e = configure_shared_memory(inner, kInnerBytes, innerConfigured))
    return e;
  if (const cudaError_t e = configure_shared_memory(outer, sizeof(OuterShared<W>), outerConfigured))
    return e;
  const int64_t blocks = (p.m + kRows - 1) / kRows, most = std::min<int64_t>(p.m, kRows);  // adapters of a block
  int64_t units = 0;
  for (int i = 0; i < (PAIR ? 1 : p.count); ++i)
    units += (p.n[i] + kUnit - 1) / kUnit;
  // What there is to do only the device knows: two CTAs an SM, or as many as could have something to do. (In the first launch of more than eight rows one of them runs at a time.)
  const int64_t items = std::clamp<int64_t>(2 * sms / kParts / blocks, 1, most * 8);
  if (const cudaError_t e = launch_kernel<2>(inner, dim3(kParts, unsigned(blocks), unsigned(items)), inner_warps(NT) * kWarp, kInnerBytes, stream, p))
    return e;
  const int64_t shares = std::clamp<int64_t>(2 * sms / blocks, 1, most * ((units + kOuterWarps - 1) / kOuterWarps));
  return launch_kernel<2>(outer, dim3(unsigned(shares), unsigned(blocks)), kOuterWarps * kWarp, sizeof(OuterShared<W>), stream, p);
}

template <class W, bool PAIR> cudaError_t launch(const AdapterParams& p, int sms, cudaStream_t stream) {
  return p.m <= 8 ? launch_blocks<W, PAIR, 1>(p, sms, stream) : launch_blocks<W, PAIR, 4>(p, sms, stream);
}

}  // namespace

cudaError_t adapters_launch(int type, bool pair, const AdapterParams& p, int sms, cudaStream_t stream) {
  switch (type) {
  case INFDEV_F32:
    return pair ? launch<float, true>(p, sms, stream) : launch<float, false>(p, sms, stream);
  case INFDEV_F16:
    return pair ? launch<__half, true>(p, sms, stream) : launch<__half, false>(p, sms, stream);
  default:
    return pair ? launch<__nv_bfloat16, true>(p, sms, stream) : launch<__nv_bfloat16, false>(p, sms, stream);
  }
}

}  // namespace infdev
