// Tables for moving pages of a cache (csrc/pages.cu): checked page ids, and the order in which copies between pages of one pool
// give what a copy from an untouched pool would. Pure functions of their arguments.
#include <pybind11/numpy.h>
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>

#include <algorithm>
#include <cstdint>
#include <numeric>
#include <stdexcept>
#include <string>
#include <tuple>
#include <vector>

namespace py = pybind11;

namespace {

void check_range(const std::vector<int64_t>& ids, int64_t num_pages) {
  for (int64_t id : ids)
    if (id < 0 || id >= num_pages) throw std::invalid_argument("page " + std::to_string(id) + " is outside the pool of " + std::to_string(num_pages));
}

py::array_t<int32_t> to_array(const std::vector<int32_t>& v) {
  py::array_t<int32_t> a(static_cast<py::ssize_t>(v.size()));
  std::copy(v.begin(), v.end(), a.mutable_data());
  return a;
}

py::array_t<int32_t> page_ids(const std::vector<int64_t>& ids, int64_t num_pages, bool unique) {
  check_range(ids, num_pages);
  if (unique) {
    std::vector<int64_t> s(ids);
    std::sort(s.begin(), s.end());
    if (std::adjacent_find(s.begin(), s.end()) != s.end()) throw std::invalid_argument("a page is named twice");
  }
  return to_array(std::vector<int32_t>(ids.begin(), ids.end()));
}

// (table, pairs, chains): table = pairs (src, dst) in order, then the chains' first pairs and the number of pairs. Within a chain no
// pair writes a page that a later one reads, except that the last pair of a cycle reads the page its first pair wrote (whose content
// the mover has kept). Chains have no page in common that either writes.
std::tuple<py::array_t<int32_t>, int, int> page_copies(const std::vector<int64_t>& src, const std::vector<int64_t>& dst, int64_t num_pages) {
  if (src.size() != dst.size()) throw std::invalid_argument("as many sources as destinations are needed");
  check_range(src, num_pages);
  check_range(dst, num_pages);
  std::vector<std::pair<int32_t, int32_t>> by_dst;                 // (dst, src)
  for (size_t i = 0; i < src.size(); ++i) by_dst.emplace_back(static_cast<int32_t>(dst[i]), static_cast<int32_t>(src[i]));
  std::sort(by_dst.begin(), by_dst.end());
  by_dst.erase(std::unique(by_dst.begin(), by_dst.end()), by_dst.end());
  for (size_t i = 1; i < by_dst.size(); ++i)
    if (by_dst[i].first == by_dst[i - 1].first) throw std::invalid_argument("page " + std::to_string(by_dst[i].first) + " has two sources");
  by_dst.erase(std::remove_if(by_dst.begin(), by_dst.end(), [](const auto& p) { return p.first == p.second; }), by_dst.end());
  const int n = static_cast<int>(by_dst.size());
  std::vector<int> parent(n), waiting(n, 0), group(n);             // parent: the pair that overwrites this pair's source
  bool overlap = false;
  for (int i = 0; i < n; ++i) {
    const auto it = std::lower_bound(by_dst.begin(), by_dst.end(), std::make_pair(by_dst[i].second, INT32_MIN));
    parent[i] = it != by_dst.end() && it->first == by_dst[i].second ? static_cast<int>(it - by_dst.begin()) : -1;
    if (parent[i] >= 0) ++waiting[parent[i]], overlap = true;
  }
  std::vector<int> order;
  order.reserve(n);
  std::iota(group.begin(), group.end(), 0);
  if (!overlap) {
    order = group;
  } else {
    auto find = [&](int i) {
      while (group[i] != i) i = group[i] = group[group[i]];
      return i;
    };
    for (int i = 0; i < n; ++i)
      if (parent[i] >= 0) group[find(i)] = find(parent[i]);
    for (int i = 0; i < n; ++i) group[i] = find(i);
    std::vector<char> done(n, 0);
    for (int i = 0; i < n; ++i)
      if (waiting[i] == 0) order.push_back(i);                     // nobody reads what this pair overwrites
    for (size_t k = 0; k < order.size(); ++k) {
      done[order[k]] = 1;
      const int p = parent[order[k]];
      if (p >= 0 && --waiting[p] == 0) order.push_back(p);
    }
    for (int i = 0; i < n; ++i)                                    // what is left are cycles
      for (int j = i; !done[j]; j = parent[j]) done[j] = 1, order.push_back(j);
  }
  std::vector<int> length(n, 0), chains;
  for (int i : order)
    if (length[group[i]]++ == 0) chains.push_back(group[i]);
  std::stable_sort(chains.begin(), chains.end(), [&](int a, int b) { return length[a] > length[b]; });   // the longest start first
  std::vector<int32_t> table(2 * n + chains.size() + 1);
  std::vector<int> at(n, 0);
  int used = 0;
  for (size_t c = 0; c < chains.size(); ++c) {
    table[2 * n + c] = used;
    at[chains[c]] = used;
    used += length[chains[c]];
  }
  table[2 * n + chains.size()] = used;
  for (int i : order) {
    const int k = at[group[i]]++;
    table[2 * k] = by_dst[i].second;
    table[2 * k + 1] = by_dst[i].first;
  }
  return {to_array(table), n, static_cast<int>(chains.size())};
}

}  // namespace

void bind_page_plan(py::module_& m) {
  m.def("page_ids", &page_ids, py::arg("ids"), py::arg("num_pages"), py::arg("unique"));
  m.def("page_copies", &page_copies, py::arg("src"), py::arg("dst"), py::arg("num_pages"));
}
