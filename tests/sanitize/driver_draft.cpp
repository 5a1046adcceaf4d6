// Sanitizer driver for the host half of the drafted-tree calls: argument checks,
// planning over many shapes, with and without host tables and within workspaces of
// every size, and the checks of host tables, whole and broken.  Built with
// AddressSanitizer and UndefinedBehaviorSanitizer on the host.  Device pointers are
// aligned dummy addresses that only a device would dereference; calls that pass their
// checks are made only where there is no GPU, so that their launch fails.  Host tables
// are heap arrays of exactly their documented sizes.  Exit status 0 on success.
#include <stdint.h>
#include <stdio.h>
#include <string.h>
#include <unistd.h>

#include <memory>
#include <random>
#include <vector>

#include "mvr_draft.h"

static int failures = 0;
#define CHECK(cond, ...)                                                                                               \
  do {                                                                                                                 \
    if (!(cond)) {                                                                                                     \
      fprintf(stderr, "FAIL %s:%d: ", __FILE__, __LINE__);                                                              \
      fprintf(stderr, __VA_ARGS__);                                                                                    \
      fprintf(stderr, " (last error: %s)\n", mvr_last_error());                                                        \
      failures++;                                                                                                      \
    }                                                                                                                  \
  } while (0)

static std::mt19937 rng(1);
static int64_t uniform(int64_t lo, int64_t hi) { return std::uniform_int_distribution<int64_t>(lo, hi)(rng); }

template <typename T = void>
static T* fake(uintptr_t k) {
  return reinterpret_cast<T*>((uintptr_t)1 << 40 | (k << 32));
}

// A heap array of exactly `n` entries (an access to the one after it is reported).
template <typename T>
struct Table {
  explicit Table(size_t n) : p(new T[n ? n : 1]()), n(n) {
    if (n == 0) p.reset();
  }
  T& operator[](size_t i) { return p[i]; }
  T* get() { return p.get(); }
  std::unique_ptr<T[]> p;
  size_t n;
};

struct Tree {
  mvr_paged_attention_args a;
  mvr_draft_trees t;
};

static Tree tree_call(int dtype, int num_seqs, int hq, int hkv, int d, int page, int max_q, int max_len) {
  Tree c;
  memset(&c, 0, sizeof c);
  c.a.dtype = dtype;
  c.a.num_seqs = num_seqs;
  c.a.num_q_heads = hq;
  c.a.num_kv_heads = hkv;
  c.a.head_dim = d;
  c.a.page_size = page;
  c.a.max_pages_per_seq = (int)(((int64_t)max_len + page - 1) / page);
  c.a.num_pages = 1 << 20;
  c.a.max_q_len = max_q;
  c.a.max_seq_len = max_len;
  c.a.q = fake(1);
  c.a.key_pool = fake(2);
  c.a.value_pool = fake(3);
  c.a.block_tables = fake<int32_t>(4);
  c.a.seq_lens = fake<int32_t>(5);
  c.a.cu_q_lens = fake<int32_t>(6);
  c.a.out = fake(7);
  c.a.q_stride_head = c.a.out_stride_head = (int64_t)num_seqs * max_q * d;
  c.a.q_stride_token = c.a.out_stride_token = d;
  c.t.masks = fake<uint32_t>(8);
  c.t.mask_words = (max_q - 1) / 32 + 1;
  return c;
}

static void check_tree_plans() {
  const int heads[][3] = {{14, 2, 64}, {28, 4, 128}, {32, 8, 128}, {8, 1, 96}, {16, 2, 256}, {4, 4, 160}, {64, 1, 32}};
  const bool no_gpu = access("/dev/kfd", F_OK) != 0;
  for (int round = 0; round < 1500; round++) {
    const int* h = heads[uniform(0, 6)];
    const int n = (int)uniform(1, round % 10 ? 40 : 600), nodes = (int)uniform(1, round % 3 ? 9 : 130);
    // (To lengths whose units are counted in coarser steps, and to the longest that a call takes.)
    const int top = round % 20 == 0 ? INT32_MAX - 1024 - nodes : (int)uniform(1, round % 4 ? 4000 : 500000);
    Tree c = tree_call((int)uniform(0, 1), n, h[0], h[1], h[2], round % 2 ? 16 : 5, nodes, top + nodes);
    Table<int32_t> sl(n), cu(n + 1);
    for (int s = 0; s < n; s++) {
      const int q = (int)uniform(round % 5 ? 1 : 0, nodes);
      cu[s + 1] = cu[s] + q;
      sl[s] = q + (int)uniform(0, top);
    }
    if (round % 7 == 0) sl[uniform(0, n - 1)] = (int)uniform(INT32_MIN, INT32_MAX); // tables that leave the bounds
    if (round % 11 == 0) cu[uniform(0, n)] = (int)uniform(-5, INT32_MAX);
    for (int hints = 0; hints < 2; hints++) {
      c.a.seq_lens_host = hints ? sl.get() : nullptr;
      c.a.cu_q_lens_host = hints ? cu.get() : nullptr;
      const size_t need = mvr_paged_attention_tree_workspace_size(&c.a, &c.t);
      CHECK(need % 256 == 0 && need < (size_t)8 << 30, "workspace of %zu bytes", need);
      if (!no_gpu || round % 10) continue;
      for (size_t bytes : {need, need / 2, (size_t)4096, (size_t)0}) {
        c.a.workspace = fake(9);
        c.a.workspace_bytes = bytes;
        CHECK(mvr_paged_attention_tree(&c.a, &c.t) == MVR_E_HIP, "a launch without a GPU");
      }
    }
  }
}

static void check_tree_tables() {
  for (int round = 0; round < 4000; round++) {
    const int n = (int)uniform(1, 5), nodes = (int)uniform(1, 70), page = (int)uniform(1, 20), top = 200;
    Tree c = tree_call(1, n, 4, 2, 64, page, nodes, top + nodes);
    c.a.num_pages = 64;
    Table<int32_t> bt((size_t)n * c.a.max_pages_per_seq), sl(n), cu(n + 1);
    for (size_t i = 0; i < bt.n; i++) bt[i] = (int)uniform(0, 63);
    for (int s = 0; s < n; s++) {
      const int q = (int)uniform(0, nodes);
      cu[s + 1] = cu[s] + q;
      sl[s] = q + (int)uniform(0, top);
    }
    c.a.total_q = round % 2 ? cu[n] : 0;
    Table<uint32_t> masks((size_t)cu[n] * c.t.mask_words);
    for (size_t i = 0; i < masks.n; i++) masks[i] = ~0u;
    auto check = [&] {
      return mvr_paged_attention_tree_validate(&c.a, &c.t, bt.get(), sl.get(), cu.get(), masks.get());
    };
    CHECK(check() == MVR_OK, "whole tables");
    switch (round % 6) { // (with a total_q the mask rows that are read lie within it)
    case 0: sl[uniform(0, n - 1)] = (int)uniform(INT32_MIN, INT32_MAX); break;
    case 1:
      if (cu[n] == 0) break; // (0: no total_q)
      c.a.total_q = cu[n];
      cu[uniform(0, n)] = (int)uniform(INT32_MIN, INT32_MAX);
      break;
    case 2: bt[uniform(0, (int64_t)bt.n - 1)] = (int)uniform(INT32_MIN, INT32_MAX); break;
    case 3: if (masks.n) masks[uniform(0, (int64_t)masks.n - 1)] = 0; break;
    }
    check();
    mvr_paged_attention_tree_validate(&c.a, &c.t, nullptr, sl.get(), nullptr, nullptr);
    mvr_paged_attention_tree_validate(&c.a, &c.t, bt.get(), nullptr, cu.get(), nullptr);
  }
}

static void check_append_tables() {
  for (int round = 0; round < 4000; round++) {
    const int n = (int)uniform(1, 5), page = (int)uniform(1, 20), top = 150;
    mvr_rope_append_args a;
    memset(&a, 0, sizeof a);
    a.dtype = (int)uniform(0, 1);
    a.num_seqs = n;
    a.num_q_heads = 4;
    a.num_kv_heads = 2;
    a.head_dim = 64;
    a.page_size = page;
    a.num_pages = 400;
    a.max_seq_len = a.rope_len = top + 20;
    a.max_pages_per_seq = (a.max_seq_len + page - 1) / page;
    a.q = a.k = a.v = fake(1);
    a.cos_table = a.sin_table = fake(2);
    a.block_tables = fake<int32_t>(3);
    a.seq_lens = fake<int32_t>(4);
    a.cu_q_lens = fake<int32_t>(5);
    a.q_out = fake(6);
    a.key_pool = fake(7);
    a.value_pool = fake(8);
    mvr_head_norms norms = {fake(9), nullptr, 1e-6f, fake<int32_t>(10)};
    Table<int32_t> sl(n), cu(n + 1), bt((size_t)n * a.max_pages_per_seq);
    for (int s = 0; s < n; s++) {
      const int q = (int)uniform(0, 20);
      cu[s + 1] = cu[s] + q;
      sl[s] = q + (int)uniform(0, top);
    }
    for (size_t i = 0; i < bt.n; i++) bt[i] = (int)(i % 400);
    a.total_q = cu[n] + (int)uniform(cu[n] == 0, 3);
    Table<int32_t> positions(a.total_q);
    Table<uint8_t> writable((size_t)a.num_pages);
    for (size_t i = 0; i < positions.n; i++) positions[i] = (int)uniform(0, a.rope_len - 1);
    for (size_t i = 0; i < writable.n; i++) writable[i] = 1;
    auto check = [&] {
      return mvr_norm_rope_append_validate(&a, &norms, bt.get(), sl.get(), cu.get(), positions.get(), writable.get());
    };
    CHECK(check() == MVR_OK || (int64_t)n * a.max_pages_per_seq > 400, "whole tables");
    switch (round % 5) {
    case 0: sl[uniform(0, n - 1)] = (int)uniform(INT32_MIN, INT32_MAX); break;
    case 1: cu[uniform(0, n)] = (int)uniform(INT32_MIN, INT32_MAX); break;
    case 2: bt[uniform(0, (int64_t)bt.n - 1)] = (int)uniform(INT32_MIN, INT32_MAX); break;
    case 3: positions[uniform(0, (int64_t)positions.n - 1)] = (int)uniform(INT32_MIN, INT32_MAX); break;
    case 4: writable[uniform(0, (int64_t)writable.n - 1)] = 0; break;
    }
    check();
    mvr_norm_rope_append_validate(&a, &norms, bt.get(), nullptr, cu.get(), nullptr, nullptr);
  }
}

static void check_compaction_tables() {
  for (int round = 0; round < 4000; round++) {
    const int n = (int)uniform(1, 4), layers = (int)uniform(1, 3), page = (int)uniform(1, 9);
    mvr_compact_drafts_args a;
    memset(&a, 0, sizeof a);
    a.dtype = (int)uniform(0, 1);
    a.num_layers = layers;
    a.num_seqs = n;
    a.num_kv_heads = 2;
    a.head_dim = 24;
    a.page_size = page;
    a.max_seq_len = 60;
    a.max_pages_per_seq = (a.max_seq_len + page - 1) / page;
    a.num_pages = (int64_t)layers * n * a.max_pages_per_seq;
    a.max_accepted = (int)uniform(1, 12);
    a.key_pool = fake(1);
    a.value_pool = fake(2);
    a.block_tables = fake<int32_t>(3);
    a.seq_lens = fake<int32_t>(4);
    a.cu_q_lens = fake<int32_t>(5);
    a.accepted = fake<int32_t>(6);
    a.accepted_lens = fake<int32_t>(7);
    a.new_seq_lens = fake<int32_t>(8);
    Table<int32_t> bt((size_t)a.num_pages), sl(n), cu(n + 1), acc((size_t)n * a.max_accepted), lens(n);
    for (size_t i = 0; i < bt.n; i++) bt[i] = (int)i;
    for (int s = 0; s < n; s++) {
      const int q = (int)uniform(0, 15);
      cu[s + 1] = cu[s] + q;
      sl[s] = q + (int)uniform(0, 40);
      int at = -1;
      for (int j = 0; j < a.max_accepted && lens[s] == j; j++) {
        at += (int)uniform(1, 3);
        if (at < q) acc[(size_t)s * a.max_accepted + lens[s]++] = at;
      }
    }
    auto check = [&] { return mvr_compact_drafts_validate(&a, bt.get(), sl.get(), cu.get(), acc.get(), lens.get()); };
    CHECK(check() == MVR_OK, "whole tables");
    switch (round % 6) {
    case 0: sl[uniform(0, n - 1)] = (int)uniform(INT32_MIN, INT32_MAX); break;
    case 1: cu[uniform(0, n)] = (int)uniform(INT32_MIN, INT32_MAX); break;
    case 2: bt[uniform(0, (int64_t)bt.n - 1)] = (int)uniform(INT32_MIN, INT32_MAX); break;
    case 3: acc[uniform(0, (int64_t)acc.n - 1)] = (int)uniform(INT32_MIN, INT32_MAX); break;
    case 4: lens[uniform(0, n - 1)] = (int)uniform(INT32_MIN, INT32_MAX); break;
    }
    check();
    mvr_compact_drafts_validate(&a, bt.get(), sl.get(), nullptr, acc.get(), lens.get());
    mvr_compact_drafts_validate(&a, bt.get(), nullptr, cu.get(), acc.get(), lens.get());
  }
}

static void check_copy_lists() {
  for (int round = 0; round < 4000; round++) {
    mvr_copy_pages_args a;
    memset(&a, 0, sizeof a);
    a.num_copies = (int)uniform(0, 6);
    a.num_kv_heads = 2;
    a.head_dim = 8;
    a.page_size = 4;
    a.num_pages = 16;
    a.key_pool = fake(1);
    a.value_pool = fake(2);
    a.src_pages = fake<int32_t>(3);
    a.dst_pages = fake<int32_t>(4);
    Table<int32_t> src(a.num_copies), dst(a.num_copies), tokens(a.num_copies);
    for (int i = 0; i < a.num_copies; i++) {
      src[i] = (int)uniform(0, 7);
      dst[i] = 8 + i;
      tokens[i] = (int)uniform(0, 4);
    }
    auto check = [&] { return mvr_copy_pages_validate(&a, src.get(), dst.get(), tokens.get()); };
    CHECK(check() == MVR_OK, "whole lists");
    if (a.num_copies) {
      Table<int32_t>& t = round % 3 == 0 ? src : round % 3 == 1 ? dst : tokens;
      t[uniform(0, a.num_copies - 1)] = (int)uniform(INT32_MIN, INT32_MAX);
      check();
    }
    mvr_copy_pages_validate(&a, nullptr, dst.get(), nullptr);
  }
}

// Scalars of every size in every field: refused or not, never undefined.
static void check_scalars() {
  auto any = [] {
    const int64_t edges[] = {0, 1, -1, 2, 7, 8, 16, 63, 64, 128, 256, 1 << 16, 1 << 26, INT32_MAX, INT32_MIN};
    return (int32_t)edges[uniform(0, 14)];
  };
  for (int round = 0; round < 20000; round++) {
    Tree c = tree_call(1, 2, 32, 8, 128, 16, 8, 1000);
    int32_t* fields[] = {&c.a.num_seqs, &c.a.num_q_heads, &c.a.num_kv_heads, &c.a.head_dim, &c.a.page_size,
                         &c.a.max_pages_per_seq, &c.a.max_q_len, &c.a.max_seq_len, &c.a.total_q, &c.t.mask_words};
    for (int k = 0; k < 3; k++) *fields[uniform(0, 9)] = any();
    if (round % 4 == 0) c.a.num_pages = (int64_t)any() * any();
    if (round % 5 == 0) c.a.sum_seq_lens = (int64_t)any() * any();
    mvr_paged_attention_tree_workspace_size(&c.a, &c.t);

    mvr_copy_pages_args p;
    memset(&p, 0, sizeof p);
    p.key_pool = p.value_pool = fake(1);
    p.num_copies = any();
    p.num_kv_heads = any();
    p.head_dim = any();
    p.page_size = any();
    p.num_pages = uniform(0, 100);
    mvr_copy_pages_validate(&p, nullptr, nullptr, nullptr);

    mvr_compact_drafts_args m;
    memset(&m, 0, sizeof m);
    m.key_pool = m.value_pool = fake(1);
    m.block_tables = m.seq_lens = m.cu_q_lens = m.accepted = m.accepted_lens = fake<int32_t>(2);
    m.new_seq_lens = fake<int32_t>(3);
    m.num_layers = any();
    m.num_seqs = any();
    m.num_kv_heads = any();
    m.head_dim = any();
    m.page_size = any();
    m.num_pages = uniform(0, 100);
    m.max_pages_per_seq = any();
    m.max_seq_len = any();
    m.max_accepted = any();
    mvr_compact_drafts_validate(&m, nullptr, nullptr, nullptr, nullptr, nullptr);

    mvr_rope_append_args r;
    memset(&r, 0, sizeof r);
    r.q = r.k = r.v = r.cos_table = r.sin_table = fake(1);
    r.block_tables = r.seq_lens = r.cu_q_lens = fake<int32_t>(2);
    r.q_out = r.key_pool = r.value_pool = fake(3);
    r.num_seqs = any();
    r.num_q_heads = any();
    r.num_kv_heads = any();
    r.head_dim = any();
    r.page_size = any();
    r.num_pages = uniform(0, 100);
    r.max_pages_per_seq = any();
    r.total_q = any();
    r.max_seq_len = any();
    r.rope_len = any();
    mvr_head_norms norms = {nullptr, nullptr, 1e-6f, round % 2 ? fake<int32_t>(4) : nullptr};
    mvr_norm_rope_append_validate(&r, &norms, nullptr, nullptr, nullptr, nullptr, nullptr);
  }
  CHECK(mvr_paged_attention_tree(nullptr, nullptr) == MVR_E_INVALID_ARGUMENT, "null structs");
  CHECK(mvr_norm_rope_append(nullptr, nullptr) == MVR_E_INVALID_ARGUMENT, "null structs");
  CHECK(mvr_compact_drafts(nullptr) == MVR_E_INVALID_ARGUMENT, "null struct");
  CHECK(mvr_copy_pages(nullptr) == MVR_E_INVALID_ARGUMENT, "null struct");
}

int main() {
  check_scalars();
  check_tree_plans();
  check_tree_tables();
  check_append_tables();
  check_compaction_tables();
  check_copy_lists();
  if (failures) return 1;
  printf("all checks passed\n");
  return 0;
}
