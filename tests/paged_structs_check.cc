// Reads the argument structs of the paged operators as a C caller's compiler lays them out (include/ops_b200.h), for a test that fills
// them from Python.
#include <cstdio>

#include "../include/ops_b200.h"

namespace {
char text[1 << 16];
int used;
template <class... A> void say(const char *fmt, A... a) { used += snprintf(text + used, sizeof(text) - (size_t)used, fmt, a...); }
void field(const char *name, const ops_layout &l, const void *base) {
  say("%s dt %u shape", name, l.dt);
  for (uint32_t i = 0; i < l.ndim; ++i) say(" %zu", l.shape[i]);
  say(" strides");
  for (uint32_t i = 0; i < l.ndim; ++i) say(" %td", l.strides[i]);
  say(" base %zx\n", (size_t)base);
}
#define FIELD(s, name) field(#name, (s)->name##_layout, (s)->name##_base)
void batch(const ops_paged_batch *b) {
  FIELD(b, page_table);
  FIELD(b, seq_start);
  FIELD(b, kv_len);
  say("max_seq %zu\n", b->max_seq);
}
}  // namespace

extern "C" {
const char *read_rope_norm(const ops_rope_norm_args *a) {
  used = 0;
  FIELD(a, y), FIELD(a, x), FIELD(a, p), FIELD(a, w);
  say("epsilon %g theta %g size %zu\n", a->epsilon, a->theta, sizeof(*a));
  return text;
}
const char *read_kv_append_paged(const ops_kv_append_paged_args *a) {
  used = 0;
  FIELD(a, q_out), FIELD(a, q), FIELD(a, k), FIELD(a, v), FIELD(a, k_pages), FIELD(a, v_pages), FIELD(a, p), FIELD(a, w);
  batch(&a->batch);
  say("epsilon %g theta %g size %zu\n", a->epsilon, a->theta, sizeof(*a));
  return text;
}
const char *read_attention_paged(const ops_attention_paged_args *a) {
  used = 0;
  FIELD(a, q), FIELD(a, k_pages), FIELD(a, v_pages), FIELD(a, o);
  batch(&a->batch);
  say("mask %u scale %g size %zu\n", (unsigned)a->mask, a->scale, sizeof(*a));
  return text;
}
}
