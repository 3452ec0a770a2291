// dh_pages: which pages of an 8-bit cache which sequence holds (include/decide_hip.h). Host memory only.
#include <algorithm>
#include <new>
#include <vector>

#include "api_internal.h"

using namespace dh_api;

struct dh_pages {
  struct Seq {
    uint64_t tokens = 0;
    std::vector<uint32_t> ids;
  };
  std::vector<uint32_t> refs;    // sequences that hold each page
  std::vector<uint64_t> unused;  // a bit per page that none holds
  uint32_t unused_count = 0;
  std::vector<Seq> seqs;

  // None of these allocates, so a call that has begun to change the tables ends.
  bool is_unused(uint32_t id) const { return unused[id / 64] >> id % 64 & 1; }
  void set_unused(uint32_t id, bool on) {
    if (is_unused(id) == on) return;
    unused[id / 64] ^= 1ull << id % 64;
    unused_count += on ? 1 : -1;
  }
  uint32_t take() {  // the lowest; there is one
    size_t w = 0;
    while (!unused[w]) ++w;
    const uint32_t id = (uint32_t)(64 * w + __builtin_ctzll(unused[w]));
    set_unused(id, false);
    refs[id] = 1;
    return id;
  }
  void drop(uint32_t id) {
    if (--refs[id] == 0) set_unused(id, true);
  }
};

namespace {
uint64_t pages_for(uint64_t tokens) { return tokens / DH_KV8_PAGE + (tokens % DH_KV8_PAGE != 0); }

// A C entry lets no C++ exception through.
template <typename F>
int guarded(const char* what, F&& f) {
  try {
    return f();
  } catch (const std::bad_alloc&) {
    return fail(DH_ENOMEM, "%s: out of host memory", what);
  } catch (...) {
    return fail(DH_EINVAL, "%s: failed", what);
  }
}
}  // namespace

extern "C" {

int dh_pages_create(uint32_t pages, uint32_t max_seqs, dh_pages** out) {
  if (!out) return fail(DH_EINVAL, "pages_create: out is null");
  if (pages < 1 || max_seqs < 1) return fail(DH_EINVAL, "pages_create: at least one page and one sequence");
  return guarded("pages_create", [&] {
    dh_pages* p = new dh_pages;
    try {
      p->refs.resize(pages);
      p->seqs.resize(max_seqs);
      p->unused.resize((pages + 63ull) / 64);
      for (uint32_t i = 0; i < pages; ++i) p->set_unused(i, true);
    } catch (...) {
      delete p;
      throw;
    }
    *out = p;
    return ok();
  });
}

void dh_pages_destroy(dh_pages* p) { delete p; }

int dh_pages_resize(dh_pages* p, uint32_t seq, uint64_t tokens, uint32_t* copy_src, uint32_t* copy_dst,
                    uint32_t* copies) {
  if (!p) return fail(DH_EINVAL, "pages_resize: null pages");
  if (seq >= p->seqs.size()) return fail(DH_EINVAL, "pages_resize: sequence %u of %zu", seq, p->seqs.size());
  if (!copy_src || !copy_dst || !copies) return fail(DH_EINVAL, "pages_resize: null pointer");
  return guarded("pages_resize", [&] {
    dh_pages::Seq& s = p->seqs[seq];
    const uint64_t want = pages_for(tokens), have = s.ids.size();
    // the page that the next token goes into, if it holds tokens already and another sequence holds it too
    const bool split = tokens > s.tokens && s.tokens % DH_KV8_PAGE != 0 && p->refs[s.ids.back()] > 1;
    const uint64_t need = (want > have ? want - have : 0) + split;
    if (need > p->unused_count)
      return fail(DH_ENOMEM, "pages_resize: %llu pages needed, %u free", (unsigned long long)need, p->unused_count);
    s.ids.reserve(want);
    *copies = 0;
    if (split) {
      *copy_src = s.ids.back();
      *copy_dst = p->take();
      *copies = 1;
      p->drop(s.ids.back());
      s.ids.back() = *copy_dst;
    }
    while (s.ids.size() < want) s.ids.push_back(p->take());
    while (s.ids.size() > want) {
      p->drop(s.ids.back());
      s.ids.pop_back();
    }
    s.tokens = tokens;
    return ok();
  });
}

int dh_pages_fork(dh_pages* p, uint32_t src, uint32_t dst, uint64_t tokens) {
  if (!p) return fail(DH_EINVAL, "pages_fork: null pages");
  if (src >= p->seqs.size() || dst >= p->seqs.size() || src == dst)
    return fail(DH_EINVAL, "pages_fork: sequences %u and %u of %zu", src, dst, p->seqs.size());
  if (!p->seqs[dst].ids.empty()) return fail(DH_EINVAL, "pages_fork: sequence %u is not empty", dst);
  if (tokens > p->seqs[src].tokens)
    return fail(DH_EINVAL, "pages_fork: %llu tokens of %llu", (unsigned long long)tokens,
                (unsigned long long)p->seqs[src].tokens);
  return guarded("pages_fork", [&] {
    const dh_pages::Seq& s = p->seqs[src];
    p->seqs[dst].ids.assign(s.ids.begin(), s.ids.begin() + (ptrdiff_t)pages_for(tokens));
    p->seqs[dst].tokens = tokens;
    for (uint32_t id : p->seqs[dst].ids) ++p->refs[id];
    return ok();
  });
}

int dh_pages_compact(dh_pages* p, uint32_t* src, uint32_t* dst, uint32_t max, uint32_t* moves) {
  if (!p) return fail(DH_EINVAL, "pages_compact: null pages");
  if (!moves || (max && (!src || !dst))) return fail(DH_EINVAL, "pages_compact: null pointer");
  return guarded("pages_compact", [&] {
    // `held` pages fill ids 0 .. held - 1 afterwards: each free id below takes the highest page above
    const uint32_t pages = (uint32_t)p->refs.size(), held = pages - p->unused_count;
    std::vector<uint32_t> from, to;
    for (uint32_t id = 0; id < held; ++id)
      if (!p->refs[id]) to.push_back(id);
    for (uint32_t id = pages; id > held && from.size() < to.size();)
      if (p->refs[--id]) from.push_back(id);
    if (from.size() > max) return fail(DH_EINVAL, "pages_compact: %zu moves, room for %u", from.size(), max);
    std::vector<uint32_t> now(pages);
    for (uint32_t id = 0; id < pages; ++id) now[id] = id;
    for (size_t i = 0; i < from.size(); ++i) {
      src[i] = from[i];
      dst[i] = to[i];
      now[from[i]] = to[i];
      p->refs[to[i]] = p->refs[from[i]];
      p->refs[from[i]] = 0;
      p->set_unused(to[i], false);
      p->set_unused(from[i], true);
    }
    for (dh_pages::Seq& s : p->seqs)
      for (uint32_t& id : s.ids) id = now[id];
    *moves = (uint32_t)from.size();
    return ok();
  });
}

int dh_pages_table(const dh_pages* p, uint32_t seq, uint64_t* tokens, uint32_t* ids, uint32_t max, uint32_t* count) {
  if (!p) return fail(DH_EINVAL, "pages_table: null pages");
  if (seq >= p->seqs.size()) return fail(DH_EINVAL, "pages_table: sequence %u of %zu", seq, p->seqs.size());
  if (!tokens || !count || (max && !ids)) return fail(DH_EINVAL, "pages_table: null pointer");
  const dh_pages::Seq& s = p->seqs[seq];
  *tokens = s.tokens;
  *count = (uint32_t)s.ids.size();
  std::copy(s.ids.begin(), s.ids.begin() + std::min<size_t>(max, s.ids.size()), ids);
  return ok();
}

uint32_t dh_pages_free(const dh_pages* p) { return p ? p->unused_count : 0; }

uint32_t dh_pages_refs(const dh_pages* p, uint32_t page) { return p && page < p->refs.size() ? p->refs[page] : 0; }

}  // extern "C"
