#include "page_pool.h"

#include <algorithm>
#include <limits>
#include <set>

namespace fo {

namespace {
// What a table and the kernels can count.
constexpr int64_t kMostTokens = std::numeric_limits<int>::max() - 1024;

at::Tensor moves_tensor(const std::vector<std::pair<int, int>>& moves) {
  at::Tensor t = at::empty({static_cast<int64_t>(moves.size()), 2}, at::kInt);
  int* at = t.data_ptr<int>();
  for (const auto& m : moves) {
    *at++ = m.first;
    *at++ = m.second;
  }
  return t;
}
}  // namespace

PagePool::PagePool(int64_t pages, int64_t page_size) : page_size_(page_size) {
  TORCH_CHECK(pages >= 0 && pages <= kMostTokens, "PagePool: number of pages out of range");
  TORCH_CHECK(page_size > 0 && page_size <= kMostTokens, "PagePool: page_size out of range");
  users_.assign(static_cast<size_t>(pages), 0);
  free_.reserve(static_cast<size_t>(pages));
  for (int64_t i = pages; i-- > 0;) free_.push_back(static_cast<int>(i));
}

const PagePool::Sequence& PagePool::At(int64_t seq) const {
  const auto it = sequences_.find(seq);
  TORCH_CHECK(it != sequences_.end(), "PagePool: no sequence ", seq);
  return it->second;
}

int PagePool::Take() {
  const int page = free_.back();
  free_.pop_back();
  users_[static_cast<size_t>(page)] = 1;
  return page;
}

void PagePool::Give(int page) {
  if (--users_[static_cast<size_t>(page)] == 0) free_.push_back(page);
}

int64_t PagePool::Add(int64_t length) {
  TORCH_CHECK(length >= 0 && length <= kMostTokens, "PagePool: length out of range");
  const int64_t need = PagesFor(length);
  TORCH_CHECK(need <= FreePages(), "PagePool: out of pages (", need, " needed, ", FreePages(), " free)");
  Sequence s;
  s.length = length;
  for (int64_t i = 0; i < need; ++i) s.pages.push_back(Take());
  sequences_.emplace(next_, std::move(s));
  return next_++;
}

void PagePool::Grow(std::vector<int64_t> seqs, std::vector<int64_t> counts) {
  TORCH_CHECK(seqs.size() == counts.size(), "PagePool: as many counts as sequences");
  int64_t need = 0;
  std::set<int64_t> seen;
  for (size_t i = 0; i < seqs.size(); ++i) {
    const Sequence& s = At(seqs[i]);
    TORCH_CHECK(seen.insert(seqs[i]).second, "PagePool: sequence ", seqs[i], " is named twice");
    TORCH_CHECK(counts[i] >= 0 && counts[i] <= kMostTokens - s.length, "PagePool: count out of range");
    need += PagesFor(s.length + counts[i]) - static_cast<int64_t>(s.pages.size());
  }
  TORCH_CHECK(need <= FreePages(), "PagePool: out of pages (", need, " needed, ", FreePages(), " free)");
  for (size_t i = 0; i < seqs.size(); ++i) {
    Sequence& s = sequences_.find(seqs[i])->second;
    s.length += counts[i];
    while (static_cast<int64_t>(s.pages.size()) < PagesFor(s.length)) s.pages.push_back(Take());
  }
}

void PagePool::Shrink(std::vector<int64_t> seqs, std::vector<int64_t> counts) {
  TORCH_CHECK(seqs.size() == counts.size(), "PagePool: as many counts as sequences");
  std::set<int64_t> seen;
  for (size_t i = 0; i < seqs.size(); ++i) {
    const Sequence& s = At(seqs[i]);
    TORCH_CHECK(seen.insert(seqs[i]).second, "PagePool: sequence ", seqs[i], " is named twice");
    TORCH_CHECK(counts[i] >= 0 && counts[i] <= s.length, "PagePool: count out of range");
    const int64_t length = s.length - counts[i];
    TORCH_CHECK(counts[i] == 0 || length % page_size_ == 0 ||
                    users_[static_cast<size_t>(s.pages[static_cast<size_t>(length / page_size_)])] == 1,
                "PagePool: sequence ", seqs[i], " would end inside a page that it shares");
  }
  for (size_t i = seqs.size(); i-- > 0;) {
    Sequence& s = sequences_.find(seqs[i])->second;
    s.length -= counts[i];
    while (static_cast<int64_t>(s.pages.size()) > PagesFor(s.length)) {
      Give(s.pages.back());
      s.pages.pop_back();
    }
  }
}

std::tuple<int64_t, at::Tensor> PagePool::Fork(int64_t seq) {
  Sequence copy = At(seq);
  std::vector<std::pair<int, int>> moves;
  if (copy.length % page_size_ != 0) {
    TORCH_CHECK(FreePages() > 0, "PagePool: out of pages (1 needed, 0 free)");
    const int from = copy.pages.back(), to = Take();
    moves.emplace_back(from, to);
    copy.pages.back() = to;
    users_[static_cast<size_t>(to)] = 0;  // counted below
  }
  for (int page : copy.pages) ++users_[static_cast<size_t>(page)];
  sequences_.emplace(next_, std::move(copy));
  return {next_++, moves_tensor(moves)};
}

void PagePool::Free(int64_t seq) {
  const Sequence& s = At(seq);
  for (auto it = s.pages.rbegin(); it != s.pages.rend(); ++it) Give(*it);
  sequences_.erase(seq);
}

at::Tensor PagePool::Compact() {
  std::vector<int> to(users_.size(), -1);
  std::vector<std::pair<int, int>> moves;
  size_t low = 0, high = users_.size();
  while (true) {
    while (low < high && users_[low] != 0) ++low;
    while (high > low && users_[high - 1] == 0) --high;
    if (low >= high) break;
    moves.emplace_back(static_cast<int>(high - 1), static_cast<int>(low));
    to[high - 1] = static_cast<int>(low);
    users_[low] = users_[high - 1];
    users_[high - 1] = 0;
  }
  for (auto& entry : sequences_) {
    for (int& page : entry.second.pages) {
      if (to[static_cast<size_t>(page)] >= 0) page = to[static_cast<size_t>(page)];
    }
  }
  free_.clear();
  for (size_t i = users_.size(); i-- > 0;) {
    if (users_[i] == 0) free_.push_back(static_cast<int>(i));
  }
  return moves_tensor(moves);
}

std::vector<int64_t> PagePool::Pages(int64_t seq) const {
  const Sequence& s = At(seq);
  return std::vector<int64_t>(s.pages.begin(), s.pages.end());
}

at::Tensor PagePool::Table(std::vector<int64_t> seqs, int64_t width) const {
  int64_t longest = 1;
  for (int64_t seq : seqs) longest = std::max(longest, static_cast<int64_t>(At(seq).pages.size()));
  TORCH_CHECK(width == 0 || width >= longest, "PagePool: a table of ", width, " pages is too narrow, ", longest, " needed");
  if (width == 0) width = longest;
  at::Tensor t = at::full({static_cast<int64_t>(seqs.size()), width}, -1, at::kInt);
  int* row = t.data_ptr<int>();
  for (int64_t seq : seqs) {
    const Sequence& s = At(seq);
    std::copy(s.pages.begin(), s.pages.end(), row);
    row += width;
  }
  return t;
}

at::Tensor PagePool::Lengths(std::vector<int64_t> seqs) const {
  at::Tensor t = at::empty({static_cast<int64_t>(seqs.size())}, at::kInt);
  int* at = t.data_ptr<int>();
  for (int64_t seq : seqs) *at++ = static_cast<int>(At(seq).length);
  return t;
}

}  // namespace fo

TORCH_LIBRARY_FRAGMENT(flashoverlap_class, m) {
  using fo::PagePool;
  m.class_<PagePool>("PagePool")
      .def(torch::init<int64_t, int64_t>())
      .def("add", &PagePool::Add)
      .def("grow", &PagePool::Grow)
      .def("shrink", &PagePool::Shrink)
      .def("fork", &PagePool::Fork)
      .def("free", &PagePool::Free)
      .def("compact", &PagePool::Compact)
      .def("length", &PagePool::Length)
      .def("pages", &PagePool::Pages)
      .def("free_pages", &PagePool::FreePages)
      .def("num_sequences", &PagePool::NumSequences)
      .def("page_size", &PagePool::PageSize)
      .def("table", &PagePool::Table)
      .def("lengths", &PagePool::Lengths);
}
