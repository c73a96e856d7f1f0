// Host side of attention over pages (paged_attention.hpp): checks, shares, workspace.
#include "paged_attention.hpp"

namespace da {

constexpr int kComputeUnits = 256;
// A sequence is one workgroup's where the table holds no more than this many tokens of it: joining costs a launch and
// sharing out a scan.  Up to 512 tokens it always pays (one sequence of 256 of 32/8 heads 6.5 instead of 9.0 us, of 512
// 9.3 and 9.1, 64 of 512 22.7 and 27.2), up to 1024 where there are workgroups for every compute unit twice (64
// sequences of 1024 42.7 and 47.0, of unlike lengths 33.9 and 36.1, but 16 of them 21.5 and 18.1); beyond, unlike lengths
// leave most of the chip waiting for the longest (64 of up to 4096 124 and 85).
constexpr int kPagedDirect = 512, kPagedDirectMany = 1024;

constexpr int64_t kPagedMostTokens = (int64_t)1 << 30;   // of a sequence: tiles ahead are counted in 32 bits

struct PagedPlan {
  int32_t groups, group_rows, shares;
  size_t prefix_bytes, border_bytes, ml_bytes, acc_bytes;
  size_t bytes() const { return shares > 1 ? prefix_bytes + border_bytes + ml_bytes + acc_bytes : 0; }
};

static int64_t paged_room(const da_paged_attention_args &r) { return (int64_t)r.pages_per_sequence * r.page_size; }

static PagedPlan paged_plan(const da_paged_attention_args &r) {
  PagedPlan p = {};
  const int rep = r.n_q_heads / r.n_kv_heads;
  const int sixteens = paged_sixteens(r.head_dim, elem_size(r.dtype), rep);
  p.group_rows = 16 * sixteens;
  p.groups = (int32_t)ceil_div(rep, p.group_rows);
  const int64_t head_groups = (int64_t)r.n_kv_heads * p.groups;
  const int64_t room = paged_room(r), units = ceil_div(room, r.dtype == DA_F32 ? 64 : 128);
  const int bytes = r.page_dtype == DA_E4M3 ? 1 : elem_size(r.dtype);
  int64_t shares = kComputeUnits * paged_resident(r.head_dim, bytes, sixteens) / head_groups;
  if (shares > units * r.n_sequences) shares = units * r.n_sequences;
  const bool many = r.n_sequences * head_groups >= 2 * kComputeUnits;
  if (room <= (many ? kPagedDirectMany : kPagedDirect) || shares <= 1) return p;
  static_assert(kComputeUnits * paged_resident(64, 1, 1) <= kPagedMostShares, "the join's threads hold that many");
  p.shares = (int32_t)shares;
  const int64_t rows = head_groups * shares * 2 * p.group_rows;
  p.prefix_bytes = (size_t)ceil_div(((int64_t)r.n_sequences + 1) * 4, 16) * 16;
  p.border_bytes = (size_t)shares * 16;
  p.ml_bytes = (size_t)rows * 2 * 4;
  p.acc_bytes = (size_t)rows * r.head_dim * 4;
  return p;
}

static int check_paged(const da_paged_attention_args &r) {
  const char *what = "da_paged_attention";
  DA_REQUIRE(r.dtype == DA_F32 || r.dtype == DA_F16 || r.dtype == DA_BF16, "%s: unknown dtype %d", what, r.dtype);
  DA_REQUIRE(r.page_dtype == r.dtype || r.page_dtype == DA_E4M3, "%s: pages of type %d for queries of type %d", what,
             r.page_dtype, r.dtype);
  if (r.page_dtype == DA_E4M3 && r.dtype == DA_F32)
    return fail(DA_ENOTSUP, "%s: 8-bit pages take 16-bit queries", what);
  DA_REQUIRE(r.n_sequences >= 0 && r.pages_per_sequence >= 0 && r.page_size > 0 && r.n_pages >= 0 && r.n_kv_heads > 0 &&
                 r.n_q_heads > 0 && r.n_q_heads % r.n_kv_heads == 0,
             "%s: bad shape", what);
  for (int t : {r.table_type, r.length_type})
    DA_REQUIRE(t == DA_I32 || t == DA_I64, "%s: unknown integer type %d", what, t);
  if (r.head_dim != 64 && r.head_dim != 96 && r.head_dim != 128 && r.head_dim != 256)
    return fail(DA_ENOTSUP, "%s: head_dim 64, 96, 128 or 256 (got %d)", what, r.head_dim);
  // (a launch counts 2^32 threads, 256 for a sequence and head; units of tokens, and shares behind them, are counted in
  // 32 bits)
  if (paged_room(r) > kPagedMostTokens || r.n_q_heads > 4096 || (int64_t)r.n_sequences * r.n_q_heads > 0xffffff ||
      r.n_sequences * (paged_room(r) / 64 + 1) > 0x7fff0000)
    return fail(DA_ENOTSUP, "%s: %d sequences of up to %lld tokens, %d heads, are too many", what, r.n_sequences,
                (long long)paged_room(r), r.n_q_heads);
  return DA_OK;
}

static bool read_args(const void *args, size_t args_bytes, da_paged_attention_args &r) {
  if (!args || args_bytes != sizeof(r)) return false;
  memcpy(&r, args, sizeof(r));
  return true;
}

}  // namespace da

extern "C" size_t da_paged_attention_workspace_bytes(const void *args, size_t args_bytes) {
  using namespace da;
  da_paged_attention_args r;
  if (!read_args(args, args_bytes, r) || check_paged(r) != DA_OK) return 0;
  return paged_plan(r).bytes();
}

extern "C" int da_paged_attention(const void *args, size_t args_bytes, void *stream) {
  using namespace da;
  da_paged_attention_args r;
  DA_REQUIRE(read_args(args, args_bytes, r), "da_paged_attention: an argument block of %d bytes", (int)sizeof(r));
  if (int rc = check_paged(r)) return rc;
  if (r.n_sequences == 0) return DA_OK;
  // (without pages or table entries no token counts, and neither is read)
  const int32_t most = r.n_pages > 0 ? (int32_t)paged_room(r) : 0;
  DA_REQUIRE(r.q && r.out && r.lengths && (!most || (r.k_pages && r.v_pages && r.page_table)),
             "da_paged_attention: null pointer");
  DA_REQUIRE(r.page_dtype == DA_E4M3 || (!r.k_scale && !r.v_scale), "da_paged_attention: scales are for 8-bit pages");
  const int e = elem_size(r.dtype), c = r.page_dtype == DA_E4M3 ? 1 : e;
  bool aligned = ((uintptr_t)r.q | (uintptr_t)r.out | (uintptr_t)r.k_pages | (uintptr_t)r.v_pages) % 16 == 0;
  for (int64_t s : r.q_strides) aligned = aligned && s * e % 16 == 0;
  for (int64_t s : r.page_strides) aligned = aligned && s * c % 16 == 0;
  DA_REQUIRE(aligned, "da_paged_attention: rows must be 16-byte aligned");
  const PagedPlan plan = paged_plan(r);
  DA_REQUIRE(plan.bytes() == 0 || (r.workspace && (uintptr_t)r.workspace % 16 == 0 &&
                                   r.workspace_bytes >= (int64_t)plan.bytes()),
             "da_paged_attention: a workspace of %lld aligned bytes", (long long)plan.bytes());
  PagedArgs a = {};
  a.q = (const char *)r.q, a.k = (const char *)r.k_pages, a.v = (const char *)r.v_pages;
  a.q_seq_b = r.q_strides[0] * e, a.q_head_b = r.q_strides[1] * e;
  a.page_b = r.page_strides[0] * c, a.tok_b = r.page_strides[1] * c, a.head_b = r.page_strides[2] * c;
  a.table = r.page_table, a.table_stride = r.table_stride, a.table64 = r.table_type;
  a.lengths = r.lengths, a.lengths64 = r.length_type;
  a.n_seqs = r.n_sequences, a.n_pages = r.n_pages, a.max_tokens = most;
  a.by_page = divisor_of(r.page_size);
  a.n_q_heads = r.n_q_heads, a.n_kv_heads = r.n_kv_heads, a.rep = r.n_q_heads / r.n_kv_heads;
  a.groups = plan.groups, a.group_rows = plan.group_rows;
  a.shares = plan.shares;
  a.scale_log2 = r.scale * kLog2e;
  a.k_scale = r.k_scale, a.v_scale = r.v_scale;
  a.out = (char *)r.out, a.lse = r.lse;
  if (plan.bytes()) {
    a.prefix = (int32_t *)r.workspace;
    a.borders = (int4 *)((char *)r.workspace + plan.prefix_bytes);
    a.part_ml = (float *)((char *)a.borders + plan.border_bytes);
    a.part_acc = (float *)((char *)a.part_ml + plan.ml_bytes);
  }
  hipStream_t s = (hipStream_t)stream;
  if (r.page_dtype == DA_E4M3)
    return r.dtype == DA_BF16 ? launch_paged<BF16, E4M3>(a, r.head_dim, s) : launch_paged<F16, E4M3>(a, r.head_dim, s);
  if (r.dtype == DA_BF16) return launch_paged<BF16, BF16>(a, r.head_dim, s);
  if (r.dtype == DA_F16) return launch_paged<F16, F16>(a, r.head_dim, s);
  return launch_paged<F32, F32>(a, r.head_dim, s);
}
