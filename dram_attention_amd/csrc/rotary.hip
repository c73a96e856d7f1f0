// Rotary positions: queries and keys turned by their tokens' positions, as tensors of their own (da_rotate,
// forward and backward) or on the way into the pages of a cache (da_paged_append).
//
//   y[a_i] = f (x[a_i] cos t - x[b_i] sin t),  y[b_i] = f (x[a_i] sin t + x[b_i] cos t),  t = position * freqs[i]
//
// for the pairs i of a head's first `rotary_dim` channels: (2i, 2i + 1) or (i, i + rotary_dim / 2).  The other
// channels are copied.  The turn's transpose is the turn by -t: the backward pass is the same kernel.
//
// Angles are formed here, in 64 bits, from a position and a frequency: a table of cosines would take 64 MiB per
// 131072 positions of a head of 128, and angles multiplied out in 32 bits are off by 2^-24 of themselves, 0.06 rad at
// the millionth position of the fastest pair.  Whole turns go away in 64 bits, then quarters of a turn, and sine and
// cosine of the rest are Taylor polynomials on |t| <= pi/4 (their next terms are below 2^-26).
//
// Bound: HBM; a row is read once and written once, up to 16 bytes a lane (16384 tokens of 32/8 heads of 128 in bf16
// 60 us = 5.6 TB/s).  A workgroup takes a few tokens: its threads form their angles, about one pair each, into LDS, while
// the first rows are on their way.  Its waves then take blocks of 64 items (a load and a store each) of a token's
// head rows laid end to end, kInFlight blocks at a time; which token, tensor and block it is, is the same for the whole
// wave and left to the scalar unit.
#include "paged_math.hpp"

namespace da {

constexpr int kTurnThreads = 256;
constexpr int kTurnWaves = kTurnThreads / 64;
constexpr int kMaxPairs = 256;     // rotary_dim / 2
constexpr int kMaxTurns = 1024;    // angles of a workgroup
constexpr int kInFlight = 3;

// Head rows: of q, then of k, then (append) of v.
struct TurnArgs {
  const char *x[3];
  char *y[3];
  int64_t x_batch_b[3], x_tok_b[3], x_head_b[3];
  int64_t y_batch_b[3], y_tok_b[3], y_head_b[3];   // (y of k and v in pages: page, token, head)
  int32_t rows[3];                                 // heads
  int32_t items[3];                                // of a token
  int32_t block_end[3];                            // a token's blocks of 64 items up to and with q's, k's, v's
  Divisor by_cols;                                 // items of a row
  int32_t head_dim, rotary_dim, half;
  int32_t tokens, group;                           // of all batches; of a workgroup
  Divisor by_tokens, by_blocks, by_pairs;          // tokens of a batch, blocks of a token, pairs of a row
  const double *freqs;
  const void *positions;
  int64_t pos_batch_stride, pos_tok_stride;
  int32_t positions64;
  float factor, sign;
  // append
  const void *table, *sequences;
  int64_t table_stride;
  int32_t table64, sequences64, n_sequences, n_pages, max_tokens;
  Divisor by_page;
  const float *scale[3];                           // per kv head, or null
};

__device__ __forceinline__ void turn_of(double position, double freq, float factor, float sign, float &c, float &s) {
  double a = position * freq * 0.15915494309189535;   // turns
  a -= rint(a);
  const double quarter = rint(4.0 * a);                // -2 .. 2
  const float t = (float)((a - 0.25 * quarter) * 6.283185307179586);
  const float u = t * t;
  float sn = fmaf(u, fmaf(u, fmaf(u, fmaf(u, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), 0.f);
  sn = fmaf(t, sn, t);
  float cs = fmaf(u, fmaf(u, fmaf(u, fmaf(u, -1.f / 3628800, 1.f / 40320), -1.f / 720), 1.f / 24), -0.5f);
  cs = fmaf(u, cs, 1.f);
  const int n = (int)quarter & 3;
  const float c1 = n & 1 ? -sn : cs, s1 = n & 1 ? cs : sn;
  c = factor * (n & 2 ? -c1 : c1);
  s = factor * sign * (n & 2 ? -s1 : s1);
}

template <int kWords>
struct Words;
template <>
struct Words<1> { typedef uint32_t type; };
template <>
struct Words<2> { typedef uint32_t type __attribute__((ext_vector_type(2))); };
template <>
struct Words<4> { typedef u32x4 type; };

// A lane's kN elements as they are loaded: 16, 8 or 4 bytes, or one element.
// kStream: rows come and go by streaming loads and stores.
template <typename T, int kN, bool kStream>
struct Held {
  static constexpr int kWords = kN * T::kBytes / 4;
  typedef typename Words<kWords>::type Vec;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const char *p, int at) {
    const Vec *from = (const Vec *)(p + (int64_t)at * T::kBytes);
    const Vec v = kStream ? __builtin_nontemporal_load(from) : *from;
    memcpy(w, &v, sizeof(v));
  }
  __device__ __forceinline__ void values(float *f) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (T::kBytes == 4) {
        f[i] = as_f32(w[i]);
      } else {
        f[2 * i] = __is_same(T, BF16) ? bf16_lo(w[i]) : f16_lo(w[i]);
        f[2 * i + 1] = __is_same(T, BF16) ? bf16_hi(w[i]) : f16_hi(w[i]);
      }
    }
  }
};
template <typename T, bool kStream>
struct Held<T, 1, kStream> {
  float v;
  __device__ __forceinline__ void load(const char *p, int at) { v = load_elem<T>(p, at); }
  __device__ __forceinline__ void values(float *f) const { f[0] = v; }
};
// kN values into elements of type TC; e4m3 ones divided by the head's scale first.
template <typename TC, int kN, bool kStream>
__device__ __forceinline__ void store_row(char *p, int at, float *f, float scale) {
  if constexpr (TC::kBytes == 1) {
#pragma unroll
    for (int i = 0; i < kN; ++i) f[i] = f[i] / scale;
    if constexpr (kN >= 4) {
#pragma unroll
      for (int i = 0; i < kN; i += 4) ((uint32_t *)(p + at))[i / 4] = pack_e4m3(f + i);
    } else {
      const float some[4] = {f[0], kN == 2 ? f[kN - 1] : 0.f, 0.f, 0.f};
      const uint32_t w = pack_e4m3(some);
      if constexpr (kN == 2) *(uint16_t *)(p + at) = (uint16_t)w;
      else p[at] = (char)w;
    }
  } else if constexpr (kN == 1) {
    store_elem<TC>(p, at, f[0]);
  } else {
    constexpr int kWords = kN * TC::kBytes / 4;
    typedef typename Words<kWords>::type Vec;
    uint32_t w[kWords];
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (TC::kBytes == 4) w[i] = __builtin_bit_cast(uint32_t, f[i]);
      else w[i] = __is_same(TC, BF16) ? pack_bf16(f[2 * i], f[2 * i + 1]) : pack_f16(f[2 * i], f[2 * i + 1]);
    }
    Vec v, *to = (Vec *)(p + (int64_t)at * TC::kBytes);
    memcpy(&v, w, sizeof(v));
    if constexpr (kStream) __builtin_nontemporal_store(v, to);
    else *to = v;
  }
}

// kN: elements a load, as many as divide a row's parts (16 bytes where they do: a 20-channel turn of heads of 80 takes 4
// bytes a lane).  kPairsInside: the interleaved layout by vectors, whose pairs lie inside one; otherwise an item is
// the two vectors (or elements) of kN pairs, and behind those single ones that are copied.
template <typename T, typename TC, int kN, bool kPairsInside, bool kPaged, bool kStream>
__global__ void __launch_bounds__(kTurnThreads) rotary_rows_kernel(const TurnArgs a) {
  __shared__ float2 turns[kMaxTurns];
  __shared__ int64_t places[kTurnThreads];   // (append) byte offsets of the tokens in the pool, -1: not stored
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int first = (int)blockIdx.x * a.group, count = min(a.group, a.tokens - first);
  const int pairs = a.rotary_dim / 2;
  const int turned_cols = kPairsInside ? a.rotary_dim / kN : pairs / kN;
  const int blocks = a.by_blocks.d * count;

  // An item's first element, and the second part's (pairs that lie apart).
  auto at_a = [&](int col) {
    if (kPairsInside) return col * kN;
    if (col >= turned_cols) return a.rotary_dim + (col - turned_cols) * kN;
    return a.half ? col * kN : 2 * col;
  };
  auto at_b = [&](int col) { return a.half ? pairs + col * kN : 2 * col + 1; };

  // What a block is (the same for the wave's lanes).
  struct Block {
    int tok, w, item;   // within the workgroup's tokens; tensor; first item
    int64_t batch, in_batch;
  };
  auto block_at = [&](int j) {
    Block x;
    x.tok = divide(j, a.by_blocks);
    const int within = j - x.tok * a.by_blocks.d;
    x.w = within < a.block_end[0] ? 0 : !kPaged || within < a.block_end[1] ? 1 : 2;
    x.item = (within - (x.w ? a.block_end[x.w - 1] : 0)) * 64;
    x.batch = divide(first + x.tok, a.by_tokens);
    x.in_batch = first + x.tok - (int)x.batch * a.by_tokens.d;
    return x;
  };
  Held<T, kN, kStream> ha[kInFlight], hb[kInFlight];
  auto load = [&](const Block &x, int u) {
    const int item = x.item + lane, row = divide(item, a.by_cols), col = item - row * a.by_cols.d;
    if (item >= a.items[x.w]) return;
    const char *p = a.x[x.w] + x.batch * a.x_batch_b[x.w] + x.in_batch * a.x_tok_b[x.w] + row * a.x_head_b[x.w];
    ha[u].load(p, at_a(col));
    if (!kPairsInside && col < turned_cols) hb[u].load(p, at_b(col));
  };
  auto store = [&](const Block &x, int u) {
    const int item = x.item + lane, row = divide(item, a.by_cols), col = item - row * a.by_cols.d;
    if (item >= a.items[x.w]) return;
    float fa[kN], fb[kN];
    const bool paired = !kPairsInside && col < turned_cols;
    ha[u].values(fa);
    if (paired) hb[u].values(fb);
    if (col < turned_cols && x.w < 2) {
      const float2 *turn = turns + x.tok * pairs + col * (kPairsInside ? kN / 2 : kN);
      if constexpr (kPairsInside) {
#pragma unroll
        for (int i = 0; i < kN; i += 2) rotate_pair(fa[i], fa[i + 1], turn[i / 2].x, turn[i / 2].y);
      } else {
#pragma unroll
        for (int i = 0; i < kN; ++i) rotate_pair(fa[i], fb[i], turn[i].x, turn[i].y);
      }
    }
    if (!kPaged || x.w == 0) {
      char *d = a.y[x.w] + x.batch * a.y_batch_b[x.w] + x.in_batch * a.y_tok_b[x.w] + row * a.y_head_b[x.w];
      store_row<T, kN, kStream>(d, at_a(col), fa, 1.f);
      if (paired) store_row<T, kN, kStream>(d, at_b(col), fb, 1.f);
    } else {
      const int64_t place = places[x.tok];
      if (place < 0) return;
      char *d = a.y[x.w] + place + row * a.y_head_b[x.w];
      const float scale = TC::kBytes == 1 && a.scale[x.w] ? a.scale[x.w][row] : 1.f;
      store_row<TC, kN, kStream>(d, at_a(col), fa, scale);
      if (paired) store_row<TC, kN, kStream>(d, at_b(col), fb, scale);
    }
  };

  bool formed = false;
  // (a wave without a block still has angles to form and a barrier to reach)
  for (int j0 = wave; j0 < blocks || !formed; j0 += kInFlight * kTurnWaves) {
#pragma unroll
    for (int u = 0; u < kInFlight; ++u)
      if (j0 + u * kTurnWaves < blocks) load(block_at(j0 + u * kTurnWaves), u);
    if (!formed) {
      formed = true;
      auto position = [&](int tok) {
        const int64_t batch = divide(first + tok, a.by_tokens);
        return load_index(a.positions, a.positions64,
                          batch * a.pos_batch_stride + (first + tok - (int)batch * a.by_tokens.d) * a.pos_tok_stride);
      };
      for (int i = threadIdx.x; i < count * pairs; i += kTurnThreads) {
        const int tok = divide(i, a.by_pairs);
        float c, s;
        turn_of((double)position(tok), a.freqs[i - tok * pairs], a.factor, a.sign, c, s);
        turns[i] = make_float2(c, s);
      }
      if constexpr (kPaged) {
        if (threadIdx.x < count) {
          const int64_t pos = position(threadIdx.x);
          const int64_t seq = a.sequences ? load_index(a.sequences, a.sequences64, first + threadIdx.x)
                                          : (int64_t)(first + threadIdx.x);
          int64_t place = -1;
          if (seq >= 0 && seq < a.n_sequences && pos >= 0 && pos < a.max_tokens) {
            const int page = divide((int)pos, a.by_page);
            const int64_t number = load_index(a.table, a.table64, seq * a.table_stride + page);
            if (number >= 0 && number < a.n_pages)
              place = number * a.y_batch_b[1] + (int64_t)((int)pos - page * a.by_page.d) * a.y_tok_b[1];
          }
          places[threadIdx.x] = place;
        }
      }
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < kInFlight; ++u)
      if (j0 + u * kTurnWaves < blocks) store(block_at(j0 + u * kTurnWaves), u);
  }
}

// Workgroups that fill the chip; tokens are taken several at a time where there are more.
constexpr int kTurnGrid = 1024;

// Fills what follows from the shape, rows taken `n` elements a load.
static int shape_rows(TurnArgs &a, int64_t batch, int64_t tokens, int n, const char *what) {
  const int pairs = a.rotary_dim / 2;
  const bool inside = n > 1 && !a.half;
  const int cols = inside ? a.head_dim / n : pairs / n + (a.head_dim - a.rotary_dim) / n;
  a.by_cols = divisor_of(cols);
  int64_t blocks = 0;
  for (int i = 0; i < 3; ++i) {
    const int64_t items = (int64_t)a.rows[i] * cols;
    blocks += ceil_div(items, 64);
    if (blocks > 1 << 24) return fail(DA_ENOTSUP, "%s: %d heads of %d channels are too many", what, a.rows[i], a.head_dim);
    a.items[i] = (int32_t)items, a.block_end[i] = (int32_t)blocks;
  }
  if (tokens > 0x7fffff00 / batch)   // (counted in 32 bits, a workgroup's tokens ahead)
    return fail(DA_ENOTSUP, "%s: %lld sequences of %lld tokens are too many", what, (long long)batch, (long long)tokens);
  a.tokens = (int32_t)(batch * tokens);
  // as many tokens as there are angles for every thread, while enough workgroups are left; more only where a launch,
  // which counts 2^32 threads, would not hold them
  const int64_t most = 0xffffff;
  a.group = 1;
  while (a.group < 64 && a.group * 2 * pairs <= kMaxTurns &&
         ((a.group * 2 * pairs <= kTurnThreads && a.tokens / (a.group * 2) >= kTurnGrid) || a.tokens / a.group >= most))
    a.group *= 2;
  if (ceil_div(a.tokens, a.group) > most)
    return fail(DA_ENOTSUP, "%s: %lld sequences of %lld tokens are too many", what, (long long)batch, (long long)tokens);
  a.by_tokens = divisor_of((int32_t)tokens), a.by_blocks = divisor_of((int32_t)blocks);
  a.by_pairs = divisor_of(pairs > 1 ? pairs : 1);
  return DA_OK;
}

// Bytes read and written from which rows come and go by streaming: the last-level cache holds 256 MiB and would
// keep none of them until they are used.  16384 tokens of 32/8 heads of 128 in bf16 (320 MiB) 72 -> 62 us, prompts of
// 30 thousand tokens into pages (720 MiB) 163 -> 153; 4900 tokens of fp16 heads (58 MiB) 14 -> 20, their rows still in
// the cache.
constexpr int64_t kStreamBytes = (int64_t)256 << 20;

template <typename T, typename TC, bool kPaged>
static int launch_rows(const TurnArgs &a, int n, hipStream_t s, const char *what) {
  const dim3 grid((unsigned)ceil_div(a.tokens, a.group)), block(kTurnThreads);
  const int64_t rows = a.rows[0] + a.rows[1] + a.rows[2];
  const bool stream = rows * a.tokens * a.head_dim * 2 * T::kBytes >= kStreamBytes;
#define DA_TURN(n, inside, streaming) \
  hipLaunchKernelGGL((rotary_rows_kernel<T, TC, n, inside, kPaged, streaming>), grid, block, 0, s, a)
#define DA_TURN_LAYOUT(n, streaming)   \
  do {                                 \
    if (a.half) DA_TURN(n, false, streaming); \
    else DA_TURN(n, true, streaming);  \
  } while (0)
  if (n == T::kVec && stream) DA_TURN_LAYOUT(T::kVec, true);
  else if (n == T::kVec) DA_TURN_LAYOUT(T::kVec, false);
  else if (n == T::kVec / 2) DA_TURN_LAYOUT(T::kVec / 2, false);
  else if (n == 2) DA_TURN_LAYOUT(2, false);
  else DA_TURN(1, false, false);
#undef DA_TURN_LAYOUT
#undef DA_TURN
  return launch_status(what);
}

static int check_turn(int head_dim, int rotary_dim, int layout, int dtype, const void *freqs, const char *what) {
  DA_REQUIRE(dtype == DA_F32 || dtype == DA_F16 || dtype == DA_BF16, "%s: unknown dtype %d", what, dtype);
  DA_REQUIRE(head_dim > 0 && rotary_dim >= 0 && rotary_dim % 2 == 0 && rotary_dim <= head_dim,
             "%s: %d channels of %d cannot turn in pairs", what, rotary_dim, head_dim);
  DA_REQUIRE(layout == DA_ROTARY_INTERLEAVED || layout == DA_ROTARY_HALF, "%s: unknown layout %d", what, layout);
  DA_REQUIRE(freqs || rotary_dim == 0, "%s: null pointer", what);
  if (rotary_dim / 2 > kMaxPairs || head_dim > 65536)
    return fail(DA_ENOTSUP, "%s: up to %d channels that turn, heads of up to 65536", what, 2 * kMaxPairs);
  return DA_OK;
}
// The most elements a load, at most 16 bytes and a power of two, that divide everything in `parts` (elements).
static int elements_a_load(int vec, int64_t parts) {
  int n = vec;
  while (n > 1 && parts % n != 0) n /= 2;
  return n;
}

}  // namespace da

extern "C" int da_rotate(const void *args, size_t args_bytes, void *stream) {
  using namespace da;
  DA_REQUIRE(args && args_bytes == sizeof(da_rotate_args), "da_rotate: an argument block of %d bytes",
             (int)sizeof(da_rotate_args));
  da_rotate_args r;
  memcpy(&r, args, sizeof(r));
  if (int rc = check_turn(r.head_dim, r.rotary_dim, r.layout, r.dtype, r.freqs, "da_rotate")) return rc;
  DA_REQUIRE(r.batch >= 0 && r.tokens >= 0 && r.n_q_heads >= 0 && r.n_k_heads >= 0 && r.n_q_heads <= 1 << 20 &&
                 r.n_k_heads <= 1 << 20,
             "da_rotate: bad shape");
  DA_REQUIRE(r.position_type == DA_I32 || r.position_type == DA_I64, "da_rotate: unknown position type %d",
             r.position_type);
  if (r.batch == 0 || r.tokens == 0 || r.n_q_heads + r.n_k_heads == 0) return DA_OK;
  DA_REQUIRE(r.positions && (!r.n_q_heads || (r.q && r.q_out)) && (!r.n_k_heads || (r.k && r.k_out)),
             "da_rotate: null pointer");
  const int e = elem_size(r.dtype), vec = 16 / e;
  TurnArgs a = {};
  const void *x[2] = {r.q, r.k};
  void *y[2] = {r.q_out, r.k_out};
  const int64_t *xs[2] = {r.q_strides, r.k_strides}, *ys[2] = {r.q_out_strides, r.k_out_strides};
  const int32_t heads[2] = {r.n_q_heads, r.n_k_heads};
  // (what all offsets have in common is the lowest bit of their union)
  int64_t parts = r.head_dim | (r.layout ? r.rotary_dim / 2 : r.rotary_dim);
  for (int i = 0; i < 2; ++i) {
    a.x[i] = (const char *)x[i];
    a.y[i] = (char *)y[i];
    a.x_batch_b[i] = xs[i][0] * e, a.x_tok_b[i] = xs[i][1] * e, a.x_head_b[i] = xs[i][2] * e;
    a.y_batch_b[i] = ys[i][0] * e, a.y_tok_b[i] = ys[i][1] * e, a.y_head_b[i] = ys[i][2] * e;
    if (!heads[i]) continue;
    DA_REQUIRE(((uintptr_t)x[i] | (uintptr_t)y[i]) % e == 0, "da_rotate: rows must be aligned to their elements");
    parts |= (int64_t)(((uintptr_t)x[i] | (uintptr_t)y[i]) / e);
    for (int j = 0; j < 3; ++j) parts |= xs[i][j] | ys[i][j];
  }
  const int n = elements_a_load(vec, parts);
  a.rows[0] = r.n_q_heads, a.rows[1] = r.n_k_heads;
  a.head_dim = r.head_dim, a.rotary_dim = r.rotary_dim, a.half = r.layout;
  a.freqs = r.freqs, a.positions = r.positions, a.positions64 = r.position_type;
  a.pos_batch_stride = r.position_strides[0], a.pos_tok_stride = r.position_strides[1];
  a.factor = r.factor, a.sign = r.inverse ? -1.f : 1.f;
  if (int rc = shape_rows(a, r.batch, r.tokens, n, "da_rotate")) return rc;
  hipStream_t s = (hipStream_t)stream;
  if (r.dtype == DA_BF16) return launch_rows<BF16, BF16, false>(a, n, s, "da_rotate");
  if (r.dtype == DA_F16) return launch_rows<F16, F16, false>(a, n, s, "da_rotate");
  return launch_rows<F32, F32, false>(a, n, s, "da_rotate");
}

extern "C" int da_paged_append(const void *args, size_t args_bytes, void *stream) {
  using namespace da;
  DA_REQUIRE(args && args_bytes == sizeof(da_paged_append_args), "da_paged_append: an argument block of %d bytes",
             (int)sizeof(da_paged_append_args));
  da_paged_append_args r;
  memcpy(&r, args, sizeof(r));
  if (int rc = check_turn(r.head_dim, r.rotary_dim, r.layout, r.dtype, r.freqs, "da_paged_append")) return rc;
  DA_REQUIRE(r.page_dtype == r.dtype || r.page_dtype == DA_E4M3, "da_paged_append: pages of type %d for rows of type %d",
             r.page_dtype, r.dtype);
  if (r.page_dtype == DA_E4M3 && r.dtype == DA_F32)
    return fail(DA_ENOTSUP, "da_paged_append: 8-bit pages take 16-bit rows");
  DA_REQUIRE(r.n_tokens >= 0 && r.n_q_heads >= 0 && r.n_kv_heads > 0 && r.n_q_heads <= 1 << 20 && r.n_kv_heads <= 1 << 20 &&
                 r.n_sequences >= 0 && r.pages_per_sequence >= 0 && r.page_size > 0 && r.n_pages >= 0,
             "da_paged_append: bad shape");
  for (int t : {r.table_type, r.position_type, r.sequence_type})
    DA_REQUIRE(t == DA_I32 || t == DA_I64, "da_paged_append: unknown integer type %d", t);
  if (r.n_tokens == 0) return DA_OK;
  DA_REQUIRE(r.k && r.v && r.positions && (!r.n_q_heads || (r.q && r.q_out)), "da_paged_append: null pointer");
  DA_REQUIRE(r.n_pages == 0 || (r.k_pages && r.v_pages), "da_paged_append: null pointer");
  DA_REQUIRE((int64_t)r.n_sequences * r.pages_per_sequence == 0 || r.page_table, "da_paged_append: null pointer");
  DA_REQUIRE(r.sequences || r.n_tokens <= r.n_sequences, "da_paged_append: %lld tokens for %d sequences",
             (long long)r.n_tokens, r.n_sequences);
  DA_REQUIRE(r.page_dtype == DA_E4M3 || (!r.k_scale && !r.v_scale), "da_paged_append: scales are for 8-bit pages");
  const int64_t room = (int64_t)r.pages_per_sequence * r.page_size;
  if (room > (int64_t)1 << 30) return fail(DA_ENOTSUP, "da_paged_append: sequences of up to 2^30 tokens");
  const int e = elem_size(r.dtype), c = r.page_dtype == DA_E4M3 ? 1 : e, vec = 16 / e;
  TurnArgs a = {};
  const void *x[3] = {r.q, r.k, r.v};
  void *y[3] = {r.q_out, r.k_pages, r.v_pages};
  const int64_t *xs[3] = {r.q_strides, r.k_strides, r.v_strides};
  int64_t parts = r.head_dim | (r.layout ? r.rotary_dim / 2 : r.rotary_dim);
  for (int i = 0; i < 3; ++i) {
    a.x[i] = (const char *)x[i];
    a.y[i] = (char *)y[i];
    a.x_tok_b[i] = xs[i][0] * e, a.x_head_b[i] = xs[i][1] * e;
    if (i == 0) {
      a.y_tok_b[0] = r.q_out_strides[0] * e, a.y_head_b[0] = r.q_out_strides[1] * e;
      if (!r.n_q_heads) continue;
      DA_REQUIRE((uintptr_t)y[0] % e == 0, "da_paged_append: rows must be aligned to their elements");
      parts |= (int64_t)((uintptr_t)y[0] / e) | r.q_out_strides[0] | r.q_out_strides[1];
    } else {
      a.y_batch_b[i] = r.page_strides[0] * c, a.y_tok_b[i] = r.page_strides[1] * c, a.y_head_b[i] = r.page_strides[2] * c;
      DA_REQUIRE((uintptr_t)y[i] % c == 0, "da_paged_append: rows must be aligned to their elements");
      parts |= (int64_t)((uintptr_t)y[i] / c);
      for (int j = 0; j < 3; ++j) parts |= r.page_strides[j];
    }
    DA_REQUIRE((uintptr_t)x[i] % e == 0, "da_paged_append: rows must be aligned to their elements");
    parts |= (int64_t)((uintptr_t)x[i] / e) | xs[i][0] | xs[i][1];
  }
  const int n = elements_a_load(vec, parts);
  a.rows[0] = r.n_q_heads, a.rows[1] = a.rows[2] = r.n_kv_heads;
  a.head_dim = r.head_dim, a.rotary_dim = r.rotary_dim, a.half = r.layout;
  a.freqs = r.freqs, a.positions = r.positions, a.positions64 = r.position_type, a.pos_tok_stride = 1;
  a.factor = r.factor, a.sign = 1.f;
  a.table = r.page_table, a.table_stride = r.table_stride, a.table64 = r.table_type;
  a.sequences = r.sequences, a.sequences64 = r.sequence_type;
  a.n_sequences = r.n_sequences, a.n_pages = r.n_pages, a.max_tokens = (int32_t)room;
  a.by_page = divisor_of(r.page_size);
  a.scale[1] = r.k_scale, a.scale[2] = r.v_scale;
  if (int rc = shape_rows(a, 1, r.n_tokens, n, "da_paged_append")) return rc;
  hipStream_t s = (hipStream_t)stream;
  if (r.page_dtype == DA_E4M3) {
    if (r.dtype == DA_BF16) return launch_rows<BF16, E4M3, true>(a, n, s, "da_paged_append");
    return launch_rows<F16, E4M3, true>(a, n, s, "da_paged_append");
  }
  if (r.dtype == DA_BF16) return launch_rows<BF16, BF16, true>(a, n, s, "da_paged_append");
  if (r.dtype == DA_F16) return launch_rows<F16, F16, true>(a, n, s, "da_paged_append");
  return launch_rows<F32, F32, true>(a, n, s, "da_paged_append");
}
