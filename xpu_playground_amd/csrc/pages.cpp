// Which pages of a cache are in use (xpu_pages_*, include/xpu_cache.h): a
// count of holders per page. Host only.
#include "../../include/xpu_cache.h"
#include "runtime_internal.hpp"

#include <algorithm>
#include <functional>
#include <queue>
#include <vector>

using xpu::guarded;
using xpu::set_error;

struct xpu_pages {
  std::vector<uint32_t> holders;
  // the free ids, lowest first
  std::priority_queue<uint32_t, std::vector<uint32_t>, std::greater<uint32_t>> free;
};

namespace {

// Every id in use, and (releasing) held often enough for its number of
// occurrences.
int check_held(const xpu_pages *p, const uint32_t *ids, uint32_t n, const char *name, bool each_once_more) {
  if (!p || (n && !ids)) return set_error(XPU_ERR_INVALID, std::string(name) + ": null argument");
  std::vector<uint32_t> sorted(ids, ids + n);
  std::sort(sorted.begin(), sorted.end());
  for (uint32_t i = 0, run = 0; i < n; ++i) {
    run = i && sorted[i] == sorted[i - 1] ? run + 1 : 1;
    const uint32_t id = sorted[i];
    if (id >= p->holders.size() || p->holders[id] == 0)
      return set_error(XPU_ERR_INVALID, std::string(name) + ": page " + std::to_string(id) + " is not in use");
    if (each_once_more ? p->holders[id] > UINT32_MAX - run : p->holders[id] < run)
      return set_error(XPU_ERR_INVALID, std::string(name) + ": page " + std::to_string(id) + " has " +
                                            std::to_string(p->holders[id]) + " holders");
  }
  return XPU_OK;
}

}  // namespace

extern "C" {

int xpu_pages_create(uint32_t n_pages, xpu_pages **out) {
  return guarded("xpu_pages_create", [&] {
    if (!out) return set_error(XPU_ERR_INVALID, "xpu_pages_create: null output");
    *out = nullptr;
    if (!n_pages) return set_error(XPU_ERR_INVALID, "xpu_pages_create: n_pages must be positive");
    auto p = std::make_unique<xpu_pages>();
    p->holders.assign(n_pages, 0);
    std::vector<uint32_t> ids(n_pages);
    for (uint32_t i = 0; i < n_pages; ++i) ids[i] = i;
    p->free = decltype(p->free)(std::greater<uint32_t>(), std::move(ids));
    *out = p.release();
    return XPU_OK;
  });
}

void xpu_pages_destroy(xpu_pages *pages) { delete pages; }

int xpu_pages_free_count(const xpu_pages *pages, uint32_t *count) {
  return guarded("xpu_pages_free_count", [&] {
    if (!pages || !count) return set_error(XPU_ERR_INVALID, "xpu_pages_free_count: null argument");
    *count = static_cast<uint32_t>(pages->free.size());
    return XPU_OK;
  });
}

int xpu_pages_holders(const xpu_pages *pages, uint32_t id, uint32_t *count) {
  return guarded("xpu_pages_holders", [&] {
    if (!pages || !count) return set_error(XPU_ERR_INVALID, "xpu_pages_holders: null argument");
    if (id >= pages->holders.size()) return set_error(XPU_ERR_INVALID, "xpu_pages_holders: no such page");
    *count = pages->holders[id];
    return XPU_OK;
  });
}

int xpu_pages_take(xpu_pages *pages, uint32_t n, uint32_t *ids) {
  return guarded("xpu_pages_take", [&] {
    if (!pages || (n && !ids)) return set_error(XPU_ERR_INVALID, "xpu_pages_take: null argument");
    if (n > pages->free.size())
      return set_error(XPU_ERR_DEVICE, "xpu_pages_take: " + std::to_string(n) + " pages asked for, " +
                                           std::to_string(pages->free.size()) + " free");
    for (uint32_t i = 0; i < n; ++i) {
      ids[i] = pages->free.top();
      pages->free.pop();
      pages->holders[ids[i]] = 1;
    }
    return XPU_OK;
  });
}

int xpu_pages_share(xpu_pages *pages, const uint32_t *ids, uint32_t n) {
  return guarded("xpu_pages_share", [&] {
    if (int rc = check_held(pages, ids, n, "xpu_pages_share", true)) return rc;
    for (uint32_t i = 0; i < n; ++i) ++pages->holders[ids[i]];
    return XPU_OK;
  });
}

int xpu_pages_release(xpu_pages *pages, const uint32_t *ids, uint32_t n) {
  return guarded("xpu_pages_release", [&] {
    if (int rc = check_held(pages, ids, n, "xpu_pages_release", false)) return rc;
    for (uint32_t i = 0; i < n; ++i)
      if (--pages->holders[ids[i]] == 0) pages->free.push(ids[i]);
    return XPU_OK;
  });
}

int xpu_pages_own(xpu_pages *pages, uint32_t *ids, uint32_t n, uint32_t *src, uint32_t *dst, uint32_t *copies) {
  return guarded("xpu_pages_own", [&] {
    if (!copies || (n && (!src || !dst))) return set_error(XPU_ERR_INVALID, "xpu_pages_own: null argument");
    if (int rc = check_held(pages, ids, n, "xpu_pages_own", false)) return rc;
    // a page listed twice belongs to one table twice: no holder can be told from the other
    std::vector<uint32_t> sorted(ids, ids + n);
    std::sort(sorted.begin(), sorted.end());
    if (std::adjacent_find(sorted.begin(), sorted.end()) != sorted.end())
      return set_error(XPU_ERR_INVALID, "xpu_pages_own: a page is listed twice");
    const uint32_t need = static_cast<uint32_t>(
        std::count_if(ids, ids + n, [&](uint32_t id) { return pages->holders[id] > 1; }));
    if (need > pages->free.size())
      return set_error(XPU_ERR_DEVICE, "xpu_pages_own: " + std::to_string(need) + " pages needed, " +
                                           std::to_string(pages->free.size()) + " free");
    *copies = 0;
    for (uint32_t i = 0; i < n; ++i) {
      if (pages->holders[ids[i]] == 1) continue;
      --pages->holders[ids[i]];
      src[*copies] = ids[i];
      ids[i] = pages->free.top();
      pages->free.pop();
      pages->holders[ids[i]] = 1;
      dst[(*copies)++] = ids[i];
    }
    return XPU_OK;
  });
}

int xpu_pages_compact(xpu_pages *pages, uint32_t *src, uint32_t *dst, uint32_t *moves) {
  return guarded("xpu_pages_compact", [&] {
    if (!pages || !src || !dst || !moves) return set_error(XPU_ERR_INVALID, "xpu_pages_compact: null argument");
    const uint32_t n = static_cast<uint32_t>(pages->holders.size());
    const uint32_t used = n - static_cast<uint32_t>(pages->free.size());
    std::vector<uint32_t> ids;
    ids.reserve(n);  // no later push allocates
    for (uint32_t i = used; i < n; ++i) ids.push_back(i);
    decltype(pages->free) rest(std::greater<uint32_t>(), std::move(ids));
    *moves = 0;
    for (uint32_t to = 0, from = used; to < used; ++to) {
      if (pages->holders[to]) continue;
      while (!pages->holders[from]) ++from;  // as many are in use past `used` as are free before it
      pages->holders[to] = pages->holders[from];
      pages->holders[from] = 0;
      src[*moves] = from;
      dst[(*moves)++] = to;
    }
    pages->free = std::move(rest);
    return XPU_OK;
  });
}

int xpu_pages_renumber(const uint32_t *src, const uint32_t *dst, uint32_t moves, uint32_t *ids, uint32_t n) {
  return guarded("xpu_pages_renumber", [&] {
    if ((moves && (!src || !dst)) || (n && !ids))
      return set_error(XPU_ERR_INVALID, "xpu_pages_renumber: null argument");
    std::vector<std::pair<uint32_t, uint32_t>> map(moves);
    for (uint32_t i = 0; i < moves; ++i) map[i] = {src[i], dst[i]};
    std::sort(map.begin(), map.end());
    for (uint32_t i = 0; i < n; ++i) {
      const auto at = std::lower_bound(map.begin(), map.end(), std::pair<uint32_t, uint32_t>{ids[i], 0});
      if (at != map.end() && at->first == ids[i]) ids[i] = at->second;
    }
    return XPU_OK;
  });
}

}  // extern "C"
