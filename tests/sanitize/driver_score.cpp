// Sanitizer driver for the host half of the calls on scores: argument checks on
// scalars of every size, planning over many shapes, with and without host tables and
// within workspaces of every size, and the checks of host tables, whole and broken.
// Built with AddressSanitizer and UndefinedBehaviorSanitizer on the host.  Device
// pointers are aligned dummy addresses that only a device would dereference; calls that
// pass their checks are made only where there is no GPU, so that their launch fails.
// Host tables are heap arrays of exactly their documented sizes.  Exit status 0 on
// success.
#include <stdint.h>
#include <stdio.h>
#include <string.h>
#include <unistd.h>

#include <memory>
#include <random>

#include "mvr_score.h"

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
static int32_t any() { return (int32_t)uniform(INT32_MIN, INT32_MAX); }

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
  T& some() { return p[uniform(0, (int64_t)n - 1)]; }
  T* get() { return p.get(); }
  std::unique_ptr<T[]> p;
  size_t n;
};

struct Scored {
  mvr_paged_attention_args a;
  mvr_score_rules r;
  mvr_key_weights w;
};

static Scored scored_call(int dtype, int num_seqs, int hq, int hkv, int d, int page, int max_q, int max_len) {
  Scored c;
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
  c.r.lse = fake<float>(8);
  c.r.lse_stride_head = (int64_t)num_seqs * max_q;
  c.w.weights = fake<float>(9);
  c.w.decay = 1;
  return c;
}

static void check_plans() {
  const int heads[][3] = {{14, 2, 64}, {28, 4, 128}, {32, 8, 128}, {8, 1, 96}, {16, 2, 256}, {4, 4, 160}, {64, 1, 32}};
  const bool no_gpu = access("/dev/kfd", F_OK) != 0;
  for (int round = 0; round < 1500; round++) {
    const int* h = heads[uniform(0, 6)];
    const int n = (int)uniform(1, round % 10 ? 40 : 600), most = (int)uniform(1, round % 3 ? 9 : 3000);
    const int top = round % 20 == 0 ? INT32_MAX - 1024 - most : (int)uniform(1, round % 4 ? 4000 : 500000);
    Scored c = scored_call((int)uniform(0, 1), n, h[0], h[1], h[2], round % 2 ? 16 : 5, most, top + most);
    c.r.cap = round % 3 ? 0.f : round % 2 ? 1e-20f : 50.f;
    c.r.window = round % 4 ? 0 : (int)uniform(1, round % 8 ? 5000 : INT32_MAX);
    if (round % 5 == 0) c.r.prefix_lens = fake<int32_t>(10);
    Table<int32_t> sl(n), cu(n + 1);
    for (int s = 0; s < n; s++) {
      const int q = (int)uniform(round % 5 ? 1 : 0, most);
      cu[s + 1] = cu[s] + q;
      sl[s] = q + (int)uniform(0, top);
    }
    if (round % 7 == 0) sl.some() = any(); // tables that leave the bounds
    if (round % 11 == 0) cu.some() = any();
    for (int hints = 0; hints < 2; hints++) {
      c.a.seq_lens_host = hints ? sl.get() : nullptr;
      c.a.cu_q_lens_host = hints ? cu.get() : nullptr;
      const size_t need = mvr_paged_attention_scored_workspace_size(&c.a, &c.r);
      CHECK(need % 256 == 0 && need < (size_t)64 << 30, "workspace of %zu bytes", need);
      if (!no_gpu || round % 10) continue;
      for (size_t bytes : {need, need / 2, (size_t)4096, (size_t)0}) {
        c.a.workspace = fake(11);
        c.a.workspace_bytes = bytes;
        const int rc = mvr_paged_attention_scored(&c.a, &c.r); // (or more than one call takes)
        CHECK(rc == MVR_E_HIP || rc == MVR_E_UNSUPPORTED, "a launch without a GPU");
        c.a.workspace = nullptr;
      }
      const int rc = mvr_attention_weights(&c.a, &c.r, &c.w);
      CHECK(rc == MVR_E_HIP || rc == MVR_E_UNSUPPORTED, "a launch without a GPU");
    }
  }
}

// Scalars of every size: refused, or planned.
static void check_scalars() {
  for (int round = 0; round < 20000; round++) {
    Scored c = scored_call(1, 4, 8, 2, 64, 16, 3, 500);
    int32_t* const fields[] = {&c.a.dtype,     &c.a.num_seqs,  &c.a.num_q_heads, &c.a.num_kv_heads, &c.a.head_dim,
                               &c.a.page_size, &c.a.max_q_len, &c.a.max_seq_len, &c.a.max_pages_per_seq, &c.a.total_q,
                               &c.r.window};
    for (int k = 0; k < 2; k++) *fields[uniform(0, 10)] = uniform(0, 1) ? any() : (int32_t)uniform(-2, 300);
    if (round % 3 == 0) c.a.num_pages = uniform(INT64_MIN, INT64_MAX);
    if (round % 5 == 0) c.r.cap = __builtin_bit_cast(float, any());
    if (round % 7 == 0) c.r.lse_stride_head = uniform(INT64_MIN, INT64_MAX);
    mvr_paged_attention_scored_workspace_size(&c.a, &c.r);
    mvr_paged_attention_scored_validate(&c.a, &c.r, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr);
    mvr_attention_weights_validate(&c.a, &c.r, &c.w, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr);
  }
}

static void check_tables() {
  for (int round = 0; round < 4000; round++) {
    const int n = (int)uniform(1, 5), most = (int)uniform(1, 70), page = (int)uniform(1, 20), top = 200;
    Scored c = scored_call(1, n, 4, 2, 64, page, most, top + most);
    c.a.num_pages = (int64_t)n * c.a.max_pages_per_seq;
    Table<int32_t> bt((size_t)n * c.a.max_pages_per_seq), sl(n), cu(n + 1), prefix(n), fresh(n);
    Table<float> slopes(4);
    for (size_t i = 0; i < bt.n; i++) bt[i] = (int)i;
    for (int s = 0; s < n; s++) {
      const int q = (int)uniform(0, most);
      cu[s + 1] = cu[s] + q;
      sl[s] = q + (int)uniform(0, top);
    }
    c.a.total_q = round % 2 ? cu[n] : 0;
    Table<int32_t> first(cu[n]);
    auto check = [&] {
      const int one = mvr_paged_attention_scored_validate(&c.a, &c.r, bt.get(), sl.get(), cu.get(), first.get(),
                                                          prefix.get(), slopes.get());
      const int two = mvr_attention_weights_validate(&c.a, &c.r, &c.w, bt.get(), sl.get(), cu.get(), first.get(),
                                                     prefix.get(), slopes.get(), fresh.get());
      return one ? one : two;
    };
    CHECK(check() == MVR_OK, "whole tables");
    switch (round % 7) { // (with a total_q the first keys that are read lie within it)
    case 0: sl.some() = any(); break;
    case 1:
      if (cu[n] == 0) break; // (0: no total_q)
      c.a.total_q = cu[n];
      cu.some() = any();
      break;
    case 2: bt.some() = any(); break;
    case 3: if (first.n) first.some() = any(); break;
    case 4: prefix.some() = any(); break;
    case 5: fresh.some() = any(); break;
    case 6: slopes.some() = __builtin_bit_cast(float, any()); break;
    }
    check();
    mvr_paged_attention_scored_validate(&c.a, &c.r, nullptr, sl.get(), nullptr, nullptr, prefix.get(), nullptr);
    mvr_attention_weights_validate(&c.a, &c.r, &c.w, bt.get(), nullptr, cu.get(), nullptr, nullptr, nullptr, nullptr);
  }
}

static void check_selections() {
  for (int round = 0; round < 4000; round++) {
    const int n = (int)uniform(1, 4), layers = (int)uniform(1, 3), page = (int)uniform(1, 9);
    mvr_select_tokens_args a;
    memset(&a, 0, sizeof a);
    a.num_layers = layers;
    a.num_seqs = n;
    a.num_kv_heads = 2;
    a.page_size = page;
    a.max_seq_len = 60;
    a.max_pages_per_seq = (a.max_seq_len + page - 1) / page;
    a.num_pages = (int64_t)layers * n * a.max_pages_per_seq;
    a.max_moves = 30;
    a.recent = (int)uniform(0, 5);
    a.first = (int)uniform(0, 5);
    a.weights = fake<float>(1);
    a.positions = fake<int32_t>(2);
    a.block_tables = fake<int32_t>(3);
    a.seq_lens = fake<int32_t>(4);
    a.next_positions = fake<int32_t>(5);
    a.kept_lens = fake<int32_t>(6);
    a.keep_lens = fake<int32_t>(7);
    a.moves = fake<int32_t>(8);
    a.num_moves = fake<int32_t>(9);
    a.new_seq_lens = fake<int32_t>(10);
    Table<int32_t> bt((size_t)a.num_pages), sl(n), next(n), kept(n), keep(n);
    for (size_t i = 0; i < bt.n; i++) bt[i] = (int)i;
    for (int s = 0; s < n; s++) {
      sl[s] = (int)uniform(0, 60);
      next[s] = sl[s] + (int)uniform(0, 1000);
      kept[s] = (int)uniform(0, sl[s]);
      keep[s] = (int)uniform(a.recent + a.first, 70);
    }
    auto check = [&] {
      return mvr_select_tokens_validate(&a, bt.get(), sl.get(), next.get(), kept.get(), keep.get());
    };
    CHECK(check() == MVR_OK, "whole tables");
    switch (round % 6) {
    case 0: sl.some() = any(); break;
    case 1: next.some() = any(); break;
    case 2: kept.some() = any(); break;
    case 3: keep.some() = any(); break;
    case 4: bt.some() = any(); break;
    case 5: (&a.max_moves)[uniform(0, 2)] = any(); break; // (recent, first)
    }
    check();
    mvr_select_tokens_validate(&a, bt.get(), nullptr, next.get(), nullptr, keep.get());
  }
}

static void check_moves() {
  for (int round = 0; round < 4000; round++) {
    const int n = (int)uniform(1, 4), layers = (int)uniform(1, 3), page = (int)uniform(1, 9);
    mvr_move_tokens_args a;
    memset(&a, 0, sizeof a);
    a.dtype = (int)uniform(0, 1);
    a.num_layers = layers;
    a.num_seqs = n;
    a.num_kv_heads = 2;
    a.head_dim = 24;
    a.page_size = page;
    a.max_pages_per_seq = (60 + page - 1) / page;
    a.num_pages = (int64_t)layers * n * a.max_pages_per_seq;
    a.max_moves = (int)uniform(1, 20);
    a.key_pool = fake(1);
    a.value_pool = fake(2);
    a.block_tables = fake<int32_t>(3);
    a.moves = fake<int32_t>(4);
    a.num_moves = fake<int32_t>(5);
    const size_t rows = (size_t)layers * n * 2;
    Table<int32_t> bt((size_t)a.num_pages), moves(rows * a.max_moves * 2), counts(rows);
    for (size_t i = 0; i < bt.n; i++) bt[i] = (int)i;
    for (size_t r = 0; r < rows; r++) {
      counts[r] = (int)uniform(0, a.max_moves);
      for (int j = 0; j < a.max_moves; j++) {
        moves[(r * a.max_moves + j) * 2] = 30 + j;
        moves[(r * a.max_moves + j) * 2 + 1] = j;
      }
    }
    auto check = [&] { return mvr_move_tokens_validate(&a, bt.get(), moves.get(), counts.get()); };
    CHECK(check() == MVR_OK, "whole tables");
    switch (round % 3) {
    case 0: moves.some() = round % 2 ? any() : (int)uniform(0, 60); break;
    case 1: counts.some() = any(); break;
    case 2: bt.some() = any(); break;
    }
    check();
    mvr_move_tokens_validate(&a, nullptr, moves.get(), counts.get());
    mvr_move_tokens_validate(&a, bt.get(), nullptr, counts.get());
  }
}

int main() {
  check_scalars();
  check_plans();
  check_tables();
  check_selections();
  check_moves();
  if (failures) fprintf(stderr, "%d failures\n", failures);
  if (!failures) printf("all checks passed\n");
  return failures != 0;
}
