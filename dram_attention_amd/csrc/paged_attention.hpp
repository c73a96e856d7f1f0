// Attention of one new token of every sequence of a batch over its keys and values in pages:
//
//   out[b, j] = sum_t w_t v_t / sum_t w_t,  w_t = exp(q[b, j] . k_t * scale - m),  m = the running maximum
//
// Bound: HBM (16 sequences of up to 128K tokens of 64/8 heads of 128 in bf16 714 us = 6.4 TB/s, one of 32/8 heads 88 =
// 5.8-6.1 TB/s, the first loads and the uneven end of 512 workgroups among it).  Every key and
// value is read once for all the query heads that share it, up to 32; a group's query rows are padded to 16 so that both products are 16x16 matrix instructions, which cost next to nothing beside the loads.
//
// Split: the sequences of a kv head are laid end to end, in units of a tile for each of the four waves, and every workgroup takes
// an equal share of that line, whatever the sequences' lengths: a share may be part of one sequence or hold several.
// Where the shares begin follows from the lengths, which only the device knows: every workgroup adds them up itself
// (a block scan of the batch's lengths out of the L2).  A sequence that one share holds whole is finished there; of
// the others each share leaves its sums, at most two, which paged_join_kernel joins by their maxima.
//
// Tile of a wave (16-bit products), 2 sets of 16 tokens, lane l = 16 g + c:
//   S^T (tokens x rows)  = K Q^T      K rows from global memory are the A operand: lane (g, c) holds token c
//   O^T (D x rows)      += V^T P^T    the accumulator layout of S^T (lane (g, c): tokens 4g .. 4g+3 of row c) is the
//                                     B operand as it stands, if the product's k index counts tokens in that order
// V^T is the A operand: lane (g, c) holds its 8 tokens of one channel.  A lane loads the slice of D/16 channels that is
// its own of each of its 8 tokens (whole rows per instruction) and pairs the tokens' halves up by byte permutes, 4 a
// channel, so V needs no LDS.  Weights go in as sums of 16-bit numbers (split_weights), three in bf16, so that they keep
// their bits: the matrix cores have the room.  fp32: tiles of 16 tokens, the same layouts with k = 4, nothing is rounded.
// e4m3 keys and values become 16-bit ones (exactly) in registers; their heads' scales go into the scores and the output.
//
// The K registers are loaded anew as soon as the scores are formed, the V registers as soon as they are consumed, page
// numbers a tile ahead of both: one set of registers each, always in flight, across the end of a sequence too, whose
// sums are put together (in LDS, by barriers that wait for LDS alone) while the next one's first tile arrives.
#pragma once
#include "attention_mfma.hpp"
#include "paged_math.hpp"

namespace da {

constexpr int kPagedThreads = 256;
constexpr int kPagedWaves = kPagedThreads / 64;
constexpr int kPagedMostShares = 1024;
constexpr int kDies = 8;

// Workgroups that a compute unit holds, by the registers that `sixteens` of query rows take.
constexpr int paged_resident(int head_dim, int bytes, int sixteens) {
  return sixteens > 1     ? (head_dim == 64 ? 3 : 2)
         : head_dim == 64 ? 4
         : head_dim == 96 || (head_dim == 128 && bytes == 1) ? 3
         : head_dim == 128 || bytes == 1                     ? 2
                                                             : 1;
}
// Sixteens of query rows that share a wave's keys and values, where a kv head has more: 64/2 heads of 128 over 1 GB 193
// us instead of 239 as two workgroups, 64/1 282 instead of 381.
constexpr int paged_sixteens(int head_dim, int bytes, int rep) {
  return rep > 16 && head_dim <= 128 && bytes < 4 ? 2 : 1;
}

struct PagedArgs {
  const char *q, *k, *v;
  int64_t q_seq_b, q_head_b, page_b, tok_b, head_b;
  const void *table, *lengths;
  int64_t table_stride;
  int32_t table64, lengths64;
  int32_t n_seqs, n_pages, max_tokens;
  Divisor by_page;
  int32_t n_q_heads, n_kv_heads, rep;
  int32_t groups, group_rows;                   // groups of 16 or 32 query rows of a kv head
  int32_t shares;                               // 0: a workgroup per sequence, nothing is joined
  float scale_log2;
  const float *k_scale, *v_scale;
  char *out;
  float *lse;
  float *part_acc, *part_ml;                    // [head group][share][2][row]
  int32_t *prefix;                              // units before sequence b; [n_seqs]: all
  int4 *borders;                                // [share]: the sequence that its border with the share ahead is the first
                                                // inside of (or -1), its first and end unit, units of a share
};

// How the two products take keys and values of type KV under queries of type T.
template <typename T, typename KV, int kD>
struct PagedTile {
  static constexpr bool kWide = T::kBytes == 4;          // fp32 products
  static constexpr int kSets = kWide ? 1 : 2;            // of 16 tokens
  static constexpr int kTokens = 16 * kSets;
  static constexpr int kUnit = kTokens * kPagedWaves;
  static constexpr int kSteps = kWide ? kD / 16 : kD / 32;   // 16-byte pieces of a query row a lane holds
  static constexpr int kSlice = kD / 16;                 // channels of a value row a lane holds
  static constexpr int kSliceWords = (kSlice * KV::kBytes + 3) / 4;
  static constexpr int kRowWords = kD * KV::kBytes / 16;     // dwords of a key row a lane holds
  // A lane's channels of a value row: 16 bytes (or all there are) of every 256; of 96, four out of the first 64 and two
  // out of the others.  One load of the lanes then takes whole lines.
  static __device__ __forceinline__ int channel(int r, int j) {
    if constexpr (kD == 96) return j < 4 ? 4 * r + j : 64 + 2 * r + (j - 4);
    constexpr int kPiece = kSlice < 16 / KV::kBytes ? kSlice : 16 / KV::kBytes;
    return j / kPiece * (16 * kPiece) + kPiece * r + j % kPiece;
  }
  // The first of the (8, or fp32 4) channels that piece s of a query row holds in lane group g.
  static __device__ __forceinline__ int piece(int s, int g) {
    if constexpr (kWide) return 16 * s + 4 * g;
    if constexpr (KV::kBytes == 1) return s / 2 < kD / 64 ? 64 * (s / 2) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g;
    return 32 * s + 8 * g;
  }
};

// log2(e) is in the scores already, so weights are powers of two, at most 2^kWeightBias<T>: 1, but for fp16 2^15, so that
// small weights keep their bits (those below 2^-40 of the largest are 0).  The running maximum is followed at once: a lag,
// which would spare rescaling, gains nothing here (711 to 713 us either way) and large values would overflow.
template <typename T>
constexpr float kWeightBias = 0.f;
template <>
inline constexpr float kWeightBias<F16> = 15.f;

// Two e4m3 as two elements of T, exactly: the low or high half of w.
template <typename T, bool kHigh>
__device__ __forceinline__ uint32_t widen_e4m3(uint32_t w) {
  if constexpr (__is_same(T, BF16))
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, kHigh));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, kHigh));
}

// Numbers of T that a weight is the sum of: three bf16 ones hold the 24 bits of fp32 (two left out up to 2^-15 of a weight;
// the third costs 128K tokens of heads of 128 and 16 sequences to 128K nothing, heads of 64 1-2 %, 8-bit rows 1-3 %, 32
// query rows a wave 6 %), two fp16 ones all but 1.5 * 2^-21 of a weight, as the second is at most 1.5 * 2^-10 of it,
// or 2^-40 of the largest weight, half of fp16's least step, whichever is more.
template <typename T>
constexpr int kWeightParts = __is_same(T, BF16) ? 3 : 2;

// Two weights as such sums, dword i of part i.  Every part but the last is below what is left of the weight, so that all
// are positive: an infinite value times them is infinite, where a rest of 0 or less would make NaN of it.  (So it is
// down to 2^-29 of the largest weight in fp16, 2^-100 in bf16; smaller ones may have parts that are 0.)
__device__ __forceinline__ uint32_t take_bf16_below(float &lo, float &hi) {
  const uint32_t a = __builtin_elementwise_sub_sat(__builtin_bit_cast(uint32_t, lo), 1u);
  const uint32_t b = __builtin_elementwise_sub_sat(__builtin_bit_cast(uint32_t, hi), 1u);
  lo -= as_f32(a & 0xffff0000u), hi -= as_f32(b & 0xffff0000u);
  return __builtin_amdgcn_perm(b, a, 0x07060302u);
}
template <typename T>
__device__ __forceinline__ void split_weights(float lo, float hi, uint32_t (&part)[kWeightParts<T>]) {
  if constexpr (__is_same(T, BF16)) {
    part[0] = take_bf16_below(lo, hi);
    part[1] = take_bf16_below(lo, hi);
    part[2] = pack_bf16(lo, hi);
  } else {
    constexpr float kBelow = 1.f - 1.f / 2048;
    part[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(lo * kBelow, hi * kBelow));
    part[1] = pack_f16(lo - f16_lo(part[0]), hi - f16_hi(part[0]));
  }
}

// A load of a part of a key or value row, streaming or not.
template <typename V, bool kStream>
__device__ __forceinline__ V load_part(const char *p) {
  if constexpr (kStream) return __builtin_nontemporal_load((const V *)p);
  return *(const V *)p;
}

// A barrier for what lies in LDS: loads from global memory stay in flight across it.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

__device__ __forceinline__ int sequence_length(const PagedArgs &a, int b) {
  const int64_t n = load_index(a.lengths, a.lengths64, b);
  return n < 0 ? 0 : n < a.max_tokens ? (int)n : a.max_tokens;
}

// The running maximum of a row that had tokens, but scores of -inf alone: below every other one, but no -inf, which says
// that no token counted.  (Their softmax is 0 / 0.)
constexpr float kAllMinusInf = -3.4028234663852886e38f;
// The output of a row whose weights add up to nothing.
__device__ __forceinline__ float no_weights(float m) { return m == -INFINITY ? 0.f : __builtin_nanf(""); }

// The sums of a row over a stretch of its sequence, or over all of it (`whole`: then the output).
// `out_row`: b * n_q_heads + query head.
template <typename T, typename Tile, int kJ>
__device__ __forceinline__ void write_sums(const PagedArgs &a, bool whole, int64_t out_row, int64_t part_row, int kD,
                                           int r, int j0, float m, float l, float v_scale, const float *at) {
  if (whole) {
    const float by = v_scale / l;
    char *o = a.out + out_row * kD * T::kBytes;
    float f[kJ];
#pragma unroll
    for (int j = 0; j < kJ; ++j) f[j] = l == 0.f ? no_weights(m) : at[j] * by;
    if constexpr (T::kBytes == 2) {
      uint32_t w[kJ / 2];
#pragma unroll
      for (int j = 0; j < kJ / 2; ++j) w[j] = MatrixOps<T>::pack(f[2 * j], f[2 * j + 1]);
#pragma unroll
      for (int j = 0; j < kJ / 2; ++j) ((uint32_t *)o)[Tile::channel(r, j0 + 2 * j) / 2] = w[j];
    } else {
#pragma unroll
      for (int j = 0; j < kJ; ++j) ((float *)o)[Tile::channel(r, j0 + j)] = f[j];
    }
    if (a.lse != nullptr && r == 0 && j0 == 0) a.lse[out_row] = l == 0.f ? -INFINITY : m * kLn2 + logf(l);
  } else {
    float *p = a.part_acc + part_row * kD;
#pragma unroll
    for (int j = 0; j < kJ; ++j) p[Tile::channel(r, j0 + j)] = at[j];
    if (r == 0 && j0 == 0) {
      a.part_ml[part_row * 2] = m;
      a.part_ml[part_row * 2 + 1] = l;
    }
  }
}

// kM: sixteens of query rows that share the keys and values a wave holds.
template <typename T, typename KV, int kD, bool kStream, int kM>
__global__ void __launch_bounds__(kPagedThreads, paged_resident(kD, KV::kBytes, kM)) paged_attention_kernel(const PagedArgs a) {
  using Tile = PagedTile<T, KV, kD>;
  constexpr bool kWide = Tile::kWide;
  constexpr int kSets = Tile::kSets, kTokens = Tile::kTokens, kUnit = Tile::kUnit, kSteps = Tile::kSteps;
  constexpr int kSlice = Tile::kSlice, kSliceWords = Tile::kSliceWords, kRowWords = Tile::kRowWords;
  constexpr int kHeld = 4 * kSets;                       // tokens whose scores and values a lane holds
  constexpr int kJ = kSlice > 8 ? 8 : kSlice;            // channels of a slice that are joined at a time
  constexpr int kRow = 16 * kJ + 4;                      // floats; the pad spreads rows over banks
  constexpr float kBias = kWeightBias<T>;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;

  __shared__ int64_t offsets[kPagedWaves][kTokens];
  __shared__ float sm_m[kPagedWaves][16], sm_l[kPagedWaves][16];
  __shared__ __align__(16) float sm_acc[kPagedWaves][16][kRow];
  __shared__ int place[4];

  // The kv heads of a share are neighbours; a kv head's groups of query rows read the same keys and values, so they go
  // to one die (workgroups go to the eight dies in turn) and start together.
  const int line = (a.shares == 0 ? a.n_seqs : a.shares) * a.n_kv_heads;
  const int turn = (int)(blockIdx.x / (unsigned)(kDies * a.groups)), in_turn = (int)blockIdx.x - turn * kDies * a.groups;
  const int width = min(kDies, line - turn * kDies), group = in_turn / width;
  const int at_line = turn * kDies + in_turn - group * width;
  const int share = at_line / a.n_kv_heads, h = at_line - share * a.n_kv_heads, hg = h * a.groups + group;
  const int rows = min(a.rep - 16 * kM * group, 16 * kM);
  const int64_t first_q = (int64_t)h * a.rep + 16 * kM * group;
  const float scale_log2 = a.scale_log2 * (KV::kBytes == 1 && a.k_scale ? a.k_scale[h] : 1.f);
  const float v_scale = KV::kBytes == 1 && a.v_scale ? a.v_scale[h] : 1.f;

  auto write_nothing = [&](int i) {
    for (int x = threadIdx.x; x < rows * kD; x += kPagedThreads) {
      const int64_t row = (int64_t)i * a.n_q_heads + first_q + x / kD;
      store_elem<T>(a.out, row * kD + x % kD, 0.f);
      if (a.lse != nullptr && x % kD == 0) a.lse[row] = -INFINITY;
    }
  };

  // ---- this workgroup's share: units [u, u_end) of the line, from sequence b that has `before` units ahead of it
  int b = share, before = 0, u = 0, u_end = 0;
  if (a.shares == 0) {
    if (a.max_tokens > 0) u_end = (a.max_tokens - 1) / kUnit + 1;   // (its length is looked at below)
  } else {
    int total;
    if (a.n_seqs == 1) {
      total = (sequence_length(a, 0) + kUnit - 1) / kUnit;
      b = 0;
      if (blockIdx.x == 0 && threadIdx.x == 0) a.prefix[0] = 0, a.prefix[1] = total;
    } else {
      const int per = (a.n_seqs + kPagedThreads - 1) / kPagedThreads;
      const int first = (int)threadIdx.x * per, last = min(first + per, a.n_seqs);
      int sum = 0;
      for (int i = first; i < last; ++i) sum += (sequence_length(a, i) + kUnit - 1) / kUnit;
      int upto = sum;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int other = __shfl_up(upto, d, 64);
        if (lane >= d) upto += other;
      }
      if (lane == 63) place[wave] = upto;
      __syncthreads();
      total = 0;
#pragma unroll
      for (int w = 0; w < kPagedWaves; ++w) {
        if (w < wave) upto += place[w];
        total += place[w];
      }
      __syncthreads();
      const int each = (total + a.shares - 1) / a.shares, begin = min(share * each, total);
      int at = upto - sum;
      if (blockIdx.x == 0) {   // what the join asks for
        for (int i = threadIdx.x; i < a.shares; i += kPagedThreads) a.borders[i] = make_int4(-1, 0, 0, 0);
        __syncthreads();
        for (int i = first, n = at; i < last; ++i) {
          const int end = n + (sequence_length(a, i) + kUnit - 1) / kUnit;
          a.prefix[i] = n;
          if (end > n && (n / each + 1) * each < end) a.borders[n / each + 1] = make_int4(i, n, end, each);
          n = end;
        }
        if (threadIdx.x == 0) a.prefix[a.n_seqs] = total;
      }
      if (at <= begin && begin < upto) {   // one thread, if there is anything to do
        int i = first;
        for (; i < last - 1; ++i) {
          const int n = (sequence_length(a, i) + kUnit - 1) / kUnit;
          if (at + n > begin) break;
          at += n;
        }
        place[0] = i, place[1] = at;
      }
      __syncthreads();
      b = place[0], before = place[1];
    }
    const int each = (total + a.shares - 1) / a.shares;
    u = min(share * each, total), u_end = min(u + each, total);
    // sequences without tokens, one after the other to the shares
    for (int i = share; i < a.n_seqs; i += a.shares)
      if (sequence_length(a, i) == 0) write_nothing(i);
  }
  const char *kbase = a.k + h * a.head_b, *vbase = a.v + h * a.head_b;

  // A stretch of a sequence: its units [from, to) of `units`, tokens up to t1; `before` units lie ahead of the sequence
  // on the line.  b = n_seqs: none.
  struct Stretch {
    int b, before, from, to, units, t1;
  };
  // The stretch at unit `u` of this share, in sequence b or one behind it.
  auto stretch_at = [&](int b, int before, int u) {
    Stretch x = {a.n_seqs, before, 0, 0, 0, 0};
    if (u >= u_end) return x;
    const int last = a.shares == 0 ? b + 1 : a.n_seqs;
    for (; b < last; ++b) {   // (ends even if a length changes while this runs)
      const int len = sequence_length(a, b);
      x.units = (len + kUnit - 1) / kUnit;
      if (x.units == 0) continue;
      x.b = b, x.from = u - before, x.to = min(u_end - before, x.units);
      x.t1 = min(x.to * kUnit, len);
      break;
    }
    return x;
  };
  u32x4 qv[kM][kSteps];
  auto load_query = [&](int b) {
#pragma unroll
    for (int r = 0; r < kM; ++r) {
      const int row = 16 * r + c;
      const char *qp = a.q + b * a.q_seq_b + (first_q + (row < rows ? row : 0)) * a.q_head_b;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        qv[r][s] = load16(qp + Tile::piece(s, g) * T::kBytes);
        if (row >= rows) qv[r][s] = u32x4{0, 0, 0, 0};
      }
    }
  };

  float m[kM], l[kM];
  f32x4 acc[kM][kSlice];
  uint32_t kk[kSets][kRowWords];
  uint32_t vv[kHeld][kSliceWords];
  uint32_t live = 0;   // of the tokens held: which count

  // The number of the page of the lane's token of a tile in sequence b, -1 if it is none; whatever the sequence's length.
  auto page_of = [&](int b, int tile) {
    const int t = min(tile + (lane & (kTokens - 1)), a.max_tokens - 1);
    const int64_t page = load_index(a.table, a.table64, b * a.table_stride + divide(t, a.by_page));
    return page >= 0 && page < a.n_pages ? (int)page : -1;
  };
  // Byte offsets of the tile's tokens in the pool, -1 for those that do not count, for the wave's lanes to read.
  auto publish = [&](int t1, int tile, int page) {
    const int t = tile + (lane & (kTokens - 1)), slot = t - divide(t, a.by_page) * a.by_page.d;
    if (lane < kTokens) offsets[wave][lane] = t < t1 && page >= 0 ? page * a.page_b + (int64_t)slot * a.tok_b : -1;
    __builtin_amdgcn_wave_barrier();
  };
  auto load_keys = [&]() {
#pragma unroll
    for (int s = 0; s < kSets; ++s) {
      const int64_t off = offsets[wave][16 * s + c];
      const char *p = kbase + (off < 0 ? 0 : off);
#pragma unroll
      for (int w = 0; w + 4 <= kRowWords; w += 4) {
        const u32x4 x = load_part<u32x4, kStream>(p + (w * 4 + g * 4) * 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) kk[s][w + i] = x[i];
      }
      if constexpr (kRowWords % 4 == 2) {   // (96 e4m3)
        const u32x2 x = load_part<u32x2, kStream>(p + (kRowWords - 2) * 16 + g * 8);
        kk[s][kRowWords - 2] = x[0], kk[s][kRowWords - 1] = x[1];
      }
    }
  };
  auto load_values = [&]() {
    live = 0;
#pragma unroll
    for (int x = 0; x < kHeld; ++x) {
      const int64_t off = offsets[wave][16 * (x / 4) + 4 * g + x % 4];
      live |= (off < 0 ? 0u : 1u) << x;
      const char *p = vbase + (off < 0 ? 0 : off);
      if constexpr (kD == 96) {
        if constexpr (KV::kBytes == 1) {
          vv[x][0] = load_part<uint32_t, kStream>(p + 4 * c);
          vv[x][1] = load_part<uint16_t, kStream>(p + 64 + 2 * c);
        } else if constexpr (KV::kBytes == 2) {
          const u32x2 y = load_part<u32x2, kStream>(p + 8 * c);
          vv[x][0] = y[0], vv[x][1] = y[1];
          vv[x][2] = load_part<uint32_t, kStream>(p + 128 + 4 * c);
        } else {
          const u32x4 y = load_part<u32x4, kStream>(p + 16 * c);
#pragma unroll
          for (int i = 0; i < 4; ++i) vv[x][i] = y[i];
          const u32x2 z = load_part<u32x2, kStream>(p + 256 + 8 * c);
          vv[x][4] = z[0], vv[x][5] = z[1];
        }
      } else if constexpr (kSliceWords == 1) {
        vv[x][0] = load_part<uint32_t, kStream>(p + 4 * c);
      } else if constexpr (kSliceWords == 2) {
        const u32x2 y = load_part<u32x2, kStream>(p + 8 * c);
        vv[x][0] = y[0], vv[x][1] = y[1];
      } else {
#pragma unroll
        for (int w = 0; w < kSliceWords; w += 4) {
          const u32x4 y = load_part<u32x4, kStream>(p + w * 64 + 16 * c);
#pragma unroll
          for (int i = 0; i < 4; ++i) vv[x][w + i] = y[i];
        }
      }
    }
  };

  // S^T of the tile in kk
  auto scores = [&](f32x4 (*st)[kSets]) {
#pragma unroll
    for (int s = 0; s < kSets; ++s) {
      f32x4 x[kM], y[kM];   // two chains
#pragma unroll
      for (int r = 0; r < kM; ++r) x[r] = y[r] = f32x4{0.f, 0.f, 0.f, 0.f};
      if constexpr (kWide) {
#pragma unroll
        for (int i = 0; i < 4 * kSteps; ++i)
#pragma unroll
          for (int r = 0; r < kM; ++r) {
            f32x4 &z = i & 1 ? y[r] : x[r];
            z = __builtin_amdgcn_mfma_f32_16x16x4f32(as_f32(kk[s][i]), as_f32(qv[r][i / 4][i % 4]), z, 0, 0, 0);
          }
      } else {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          u32x4 ka;
          if constexpr (KV::kBytes == 1) {
            const uint32_t w0 = kk[s][2 * i], w1 = kk[s][2 * i + 1];
            ka = u32x4{widen_e4m3<T, false>(w0), widen_e4m3<T, true>(w0), widen_e4m3<T, false>(w1),
                       widen_e4m3<T, true>(w1)};
          } else {
            ka = u32x4{kk[s][4 * i], kk[s][4 * i + 1], kk[s][4 * i + 2], kk[s][4 * i + 3]};
          }
#pragma unroll
          for (int r = 0; r < kM; ++r) {
            f32x4 &z = i & 1 ? y[r] : x[r];
            z = MatrixOps<T>::k32(ka, qv[r][i], z);
          }
        }
      }
#pragma unroll
      for (int r = 0; r < kM; ++r) st[r][s] = x[r] + y[r];
    }
  };

  // Weights of the tile's scores; O^T += V^T P^T
  auto weigh = [&](f32x4 (*st)[kSets]) {
    float p[kM][kHeld];
#pragma unroll
    for (int r = 0; r < kM; ++r) {
      float top = -INFINITY;
#pragma unroll
      for (int x = 0; x < kHeld; ++x) {
        p[r][x] = live >> x & 1 ? st[r][x / 4][x % 4] * scale_log2 : -INFINITY;
        top = fmaxf(top, p[r][x]);
      }
      if (__any(top > m[r] + kBias)) {
        float mx = top - kBias;
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(fmaxf(mx, __shfl_xor(mx, 32, 64)), m[r]);
        const float alpha = mx == -INFINITY ? 1.f : fast_exp2(m[r] - mx);
        m[r] = mx;
        l[r] *= alpha;
#pragma unroll
        for (int j = 0; j < kSlice; ++j) acc[r][j] *= alpha;
      }
      const float ref = m[r] == -INFINITY ? 0.f : m[r];
#pragma unroll
      for (int x = 0; x < kHeld; ++x) {
        p[r][x] = fast_exp2(p[r][x] - ref);
        l[r] += p[r][x];
      }
    }
    // values of tokens that do not count are memory nobody vouches for: 0 * NaN must not arise
    if (__any(live != (1u << kHeld) - 1)) {
#pragma unroll
      for (int x = 0; x < kHeld; ++x)
#pragma unroll
        for (int w = 0; w < kSliceWords; ++w) vv[x][w] = live >> x & 1 ? vv[x][w] : 0u;
    }
    if constexpr (kWide) {
#pragma unroll
      for (int x = 0; x < kHeld; ++x)
#pragma unroll
        for (int j = 0; j < kSlice; ++j)
#pragma unroll
          for (int r = 0; r < kM; ++r)
            acc[r][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(as_f32(vv[x][j]), p[r][x], acc[r][j], 0, 0, 0);
    } else {
      constexpr int kParts = kWeightParts<T>;
      u32x4 parts[kM][kParts];
#pragma unroll
      for (int r = 0; r < kM; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t part[kParts];
          split_weights<T>(p[r][2 * i], p[r][2 * i + 1], part);
#pragma unroll
          for (int n = 0; n < kParts; ++n) parts[r][n][i] = part[n];
        }
#pragma unroll
      for (int jj = 0; jj < kSlice / 2; ++jj) {   // a dword: channels 2jj, 2jj + 1 of each token
        uint32_t w[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          if constexpr (KV::kBytes == 1)
            w[x] = jj & 1 ? widen_e4m3<T, true>(vv[x][jj / 2]) : widen_e4m3<T, false>(vv[x][jj / 2]);
          else
            w[x] = vv[x][jj];
        }
        u32x4 even, odd;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          even[i] = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x05040100u);
          odd[i] = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x07060302u);
        }
#pragma unroll
        for (int n = 0; n < kParts; ++n)
#pragma unroll
          for (int r = 0; r < kM; ++r) {
            acc[r][2 * jj] = MatrixOps<T>::k32(even, parts[r][n], acc[r][2 * jj]);
            acc[r][2 * jj + 1] = MatrixOps<T>::k32(odd, parts[r][n], acc[r][2 * jj + 1]);
          }
      }
    }
  };

  // A wave's first tile of a stretch is loaded before the sums of the stretch ahead are put together.
  auto first_tile = [&](const Stretch &x) { return x.from * kUnit + wave * kTokens; };
  if (u >= u_end) {
    if (a.shares == 0) write_nothing(b);   // (a table or a pool without pages)
    return;
  }
  // (the first loads wait for no length)
  load_query(b);
  const int tile0 = (u - before) * kUnit + wave * kTokens, page0 = page_of(b, tile0);
  int next = page_of(b, tile0 + kUnit);   // page numbers of the tile behind the one that is loaded
  Stretch cur = stretch_at(b, before, u);
  if (cur.b != b) {
    if (a.shares == 0) write_nothing(b);
    return;   // (of a share: only if a length has changed since)
  }
  publish(cur.t1, tile0, page0);
  load_keys();
  load_values();
  for (;;) {
    Stretch nxt = {a.n_seqs, 0, 0, 0, 0, 0};
    if (a.shares != 0) nxt = stretch_at(cur.b + 1, cur.before + cur.units, cur.before + cur.to);
    const bool more = nxt.b < a.n_seqs;
    int page0 = -1, page1 = -1;
    if (more) {
      page0 = page_of(nxt.b, first_tile(nxt));
      page1 = page_of(nxt.b, first_tile(nxt) + kUnit);
    }
#pragma unroll
    for (int r = 0; r < kM; ++r) {
      m[r] = -INFINITY, l[r] = 0.f;
#pragma unroll
      for (int j = 0; j < kSlice; ++j) acc[r][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    int tile = first_tile(cur);
    const bool any = tile < cur.t1;
    for (; tile + kUnit < cur.t1; tile += kUnit) {
      f32x4 st[kM][kSets];
      const int page = page_of(cur.b, tile + 2 * kUnit);
      scores(st);
      publish(cur.t1, tile + kUnit, next);
      load_keys();
      weigh(st);
      load_values();
      next = page;
    }
    {
      f32x4 st[kM][kSets];
      const bool next_any = more && first_tile(nxt) < nxt.t1;
      if (any) scores(st);
      if (next_any) {
        publish(nxt.t1, first_tile(nxt), page0);
        load_keys();
      }
      if (any) weigh(st);
      if (next_any) {
        load_values();
        load_query(nxt.b);
        next = page1;
      }
    }
#pragma unroll
    for (int r = 0; r < kM; ++r) {
      l[r] += __shfl_xor(l[r], 16, 64);
      l[r] += __shfl_xor(l[r], 32, 64);
    }
    bool none = false;
#pragma unroll
    for (int r = 0; r < kM; ++r) none = none || m[r] == -INFINITY;
    if (any && __any(none)) {   // (rare: whether a token counted is looked up again rather than carried along)
      bool counted = false;
      for (int t = first_tile(cur); t < cur.t1 && !counted; t += kUnit)
        counted = __any(t + (lane & (kTokens - 1)) < cur.t1 && page_of(cur.b, t) >= 0);
#pragma unroll
      for (int r = 0; r < kM; ++r)
        if (counted) m[r] = fmaxf(m[r], kAllMinusInf);
    }

    // ---- the waves' sums together, sixteen rows and kJ channels of each slice at a time
    const bool whole = cur.from == 0 && cur.to == cur.units;
    const int64_t part = (((int64_t)hg * a.shares + share) * 2 + (cur.from == 0 ? 1 : 0)) * (16 * kM);
#pragma unroll
    for (int pass = 0; pass < kM * (kSlice / kJ); ++pass) {
      constexpr int kSlices = kSlice / kJ;
      const int mr = pass / kSlices, j0 = pass % kSlices * kJ;
      if (16 * mr >= rows) break;
      lds_barrier();   // (what the last pass or stretch left there has been read)
      if (16 * mr + c < rows) {
        if (g == 0) sm_m[wave][c] = m[mr], sm_l[wave][c] = l[mr];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < kJ; ++j) sm_acc[wave][c][(4 * g + i) * kJ + j] = acc[mr][j0 + j][i];
      }
      lds_barrier();
      const int in_pass = threadIdx.x >> 4, r = threadIdx.x & 15, row = 16 * mr + in_pass;
      if (row < rows) {
        float mx = sm_m[0][in_pass];
#pragma unroll
        for (int w = 1; w < kPagedWaves; ++w) mx = fmaxf(mx, sm_m[w][in_pass]);
        float sum = 0.f, at[kJ];
#pragma unroll
        for (int j = 0; j < kJ; ++j) at[j] = 0.f;
#pragma unroll
        for (int w = 0; w < kPagedWaves; ++w) {
          const float by = mx == -INFINITY ? 1.f : fast_exp2(sm_m[w][in_pass] - mx);
          sum += sm_l[w][in_pass] * by;
#pragma unroll
          for (int j = 0; j < kJ; ++j) at[j] += sm_acc[w][in_pass][r * kJ + j] * by;
        }
        write_sums<T, Tile, kJ>(a, whole, (int64_t)cur.b * a.n_q_heads + first_q + row, part + row, kD, r, j0, mx, sum,
                                v_scale, at);
      }
    }
    if (!more) break;
    cur = nxt;
  }
}

// The sums of sequences that more than one share holds: a workgroup for each query head and sequence or, where
// there are fewer, inner border of two shares.  Bound: its launch and three rounds to memory, one for the stretch of shares,
// one for all that they left (which waits for no weights), one for the output: every wave forms the weights for itself.
template <typename T, int kD>
__global__ void __launch_bounds__(kPagedThreads) paged_join_kernel(const PagedArgs a, const bool by_border) {
  constexpr int kLanes = kD / 4, kParts = kPagedThreads / kLanes, kAhead = 8;
  __shared__ __align__(16) float sums[kParts][kD];
  __shared__ float weight[kPagedMostShares];
  const int hq = (int)(blockIdx.x % (unsigned)a.n_q_heads), at = (int)(blockIdx.x / (unsigned)a.n_q_heads);
  const int lane = threadIdx.x & 63;
  int b = at, s0, n;
  if (by_border) {
    const int4 x = a.borders[at + 1];
    if (x.x < 0) return;
    b = x.x, s0 = at, n = (x.z - 1) / x.w - s0 + 1;
  } else {
    const int begin = a.prefix[b], end = a.prefix[b + 1], each = (a.prefix[a.n_seqs] + a.shares - 1) / a.shares;
    if (begin == end) return;
    s0 = begin / each, n = (end - 1) / each - s0 + 1;
    if (n == 1) return;
  }
  const int h = hq / a.rep, rr = hq - h * a.rep;
  const int64_t hg = (int64_t)h * a.groups + rr / a.group_rows;
  const int in_group = rr % a.group_rows;
  auto row = [&](int i) { return ((hg * a.shares + s0 + i) * 2 + (i == 0 ? 1 : 0)) * a.group_rows + in_group; };
  auto maximum_and_sum = [&](int i) {
    return i < n ? *(const float2 *)(a.part_ml + row(i) * 2) : make_float2(-INFINITY, 0.f);
  };

  const int part = threadIdx.x / kLanes, d = threadIdx.x % kLanes * 4;
  const float2 first = maximum_and_sum(lane);
  f32x4 ahead[kAhead];
#pragma unroll
  for (int t = 0; t < kAhead; ++t) {
    const int i = part + t * kParts;
    ahead[t] = part < kParts && i < n ? *(const f32x4 *)(a.part_acc + row(i) * kD + d) : f32x4{0.f, 0.f, 0.f, 0.f};
  }
  float mx = first.x;
  for (int i = lane + 64; i < n; i += 64) mx = fmaxf(mx, maximum_and_sum(i).x);
  mx = group_max<64>(mx);
  float l = 0.f;
  for (int i = lane; i < n; i += 64) {
    const float2 x = i == lane ? first : maximum_and_sum(i);
    const float by = mx == -INFINITY ? 1.f : fast_exp2(x.x - mx);
    weight[i] = by;   // (the same from every wave)
    l += x.y * by;
  }
  l = group_sum<64>(l);
  __builtin_amdgcn_wave_barrier();

  if (part < kParts) {
    f32x4 sum = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < kAhead; ++t)
      if (part + t * kParts < n) sum += ahead[t] * weight[part + t * kParts];
    for (int i = part + kAhead * kParts; i < n; i += kParts)
      sum += *(const f32x4 *)(a.part_acc + row(i) * kD + d) * weight[i];
    *(f32x4 *)&sums[part][d] = sum;
  }
  __syncthreads();
  const int64_t out_row = (int64_t)b * a.n_q_heads + hq;
  const float v_scale = a.v_scale ? a.v_scale[h] : 1.f;
  for (int x = threadIdx.x; x < kD; x += kPagedThreads) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < kParts; ++i) t += sums[i][x];
    store_elem<T>(a.out, out_row * kD + x, l == 0.f ? no_weights(mx) : t * (v_scale / l));
  }
  if (threadIdx.x == 0 && a.lse != nullptr) a.lse[out_row] = l == 0.f ? -INFINITY : mx * kLn2 + logf(l);
}

// Defined per pair of types in paged_attention_*.hip.
template <typename T, typename KV>
int launch_paged(const PagedArgs &a, int head_dim, hipStream_t s);
template <> int launch_paged<BF16, BF16>(const PagedArgs &, int, hipStream_t);
template <> int launch_paged<F16, F16>(const PagedArgs &, int, hipStream_t);
template <> int launch_paged<F32, F32>(const PagedArgs &, int, hipStream_t);
template <> int launch_paged<BF16, E4M3>(const PagedArgs &, int, hipStream_t);
template <> int launch_paged<F16, E4M3>(const PagedArgs &, int, hipStream_t);

template <typename T, typename KV, int kD>
int launch_paged_dim(const PagedArgs &a, hipStream_t s) {
  const unsigned head_groups = (unsigned)(a.n_kv_heads * a.groups);
  const unsigned blocks = head_groups * (unsigned)(a.shares == 0 ? a.n_seqs : a.shares);
  // Keys and values that are read once come by streaming where their rows are whole lines: 141 instead of 153 us for 800 MB
  // of e4m3 rows of 128, 94 instead of 104 for 128K tokens of bf16 ones, 146 instead of 152 for 800 MB of fp32 ones (of 256
  // 295 instead of 285 for 1.6 GB).  Rows that share lines are read faster through the caches (bf16 ones of 96: 223 instead
  // of 261 us for 1.2 GB, e4m3 ones of 64: 206, 236), and so are those that several groups of query heads read (two of 32
  // of 64/1 heads of 128: 282 instead of 327).  (All from one run.)
  constexpr bool kWholeLines = kD * KV::kBytes % 128 == 0;
  const bool stream = kWholeLines && a.groups == 1;
#define DA_PAGED(streaming, sixteens)                                                                              \
  hipLaunchKernelGGL((paged_attention_kernel<T, KV, kD, streaming, sixteens>), dim3(blocks), dim3(kPagedThreads), 0, s, a)
  constexpr int kMost = paged_sixteens(kD, T::kBytes, 32);
  if (a.group_rows > 16 && stream) DA_PAGED(kWholeLines, kMost);
  else if (a.group_rows > 16) DA_PAGED(false, kMost);
  else if (stream) DA_PAGED(kWholeLines, 1);
  else DA_PAGED(false, 1);
#undef DA_PAGED
  if (a.shares > 1) {
    const bool by_border = a.shares - 1 < a.n_seqs;
    const unsigned joins = (unsigned)a.n_q_heads * (unsigned)(by_border ? a.shares - 1 : a.n_seqs);
    hipLaunchKernelGGL((paged_join_kernel<T, kD>), dim3(joins), dim3(kPagedThreads), 0, s, a, by_border);
  }
  return launch_status("da_paged_attention");
}

#define DA_PAGED_TYPES(T, KV)                                                         \
  template <>                                                                         \
  int launch_paged<T, KV>(const PagedArgs &a, int head_dim, hipStream_t s) {          \
    switch (head_dim) {                                                               \
      case 64: return launch_paged_dim<T, KV, 64>(a, s);                              \
      case 96: return launch_paged_dim<T, KV, 96>(a, s);                              \
      case 128: return launch_paged_dim<T, KV, 128>(a, s);                            \
      default: return launch_paged_dim<T, KV, 256>(a, s);                             \
    }                                                                                 \
  }

}  // namespace da
