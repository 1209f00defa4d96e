// Which pages of a key-value cache belong to which sequence: host bookkeeping, without a GPU.
//
// A sequence is a length and a list of pages; all but the last are full.  Full pages are never written again, so a fork
// shares them (counted), and copies only a last page that is not full.  Operations that cannot be done leave everything as
// it was and throw.  Not for several threads at once.
#pragma once

#include <torch/custom_class.h>
#include <torch/torch.h>

#include <map>
#include <tuple>
#include <vector>

namespace fo {

class PagePool : public torch::CustomClassHolder {
 public:
  PagePool(int64_t pages, int64_t page_size);
  // A new sequence of `length` tokens, with pages for them.
  int64_t Add(int64_t length);
  // Tokens behind the last ones: sequence seqs[i] becomes counts[i] longer.  All of them or none.
  void Grow(std::vector<int64_t> seqs, std::vector<int64_t> counts);
  // Takes back the last counts[i] tokens of sequence seqs[i], and the pages behind them.  All of them or none; a sequence does
  // not come to end inside a page that it shares, which its next tokens would change for the others.  What Grow has just done
  // is undone to the last free page.
  void Shrink(std::vector<int64_t> seqs, std::vector<int64_t> counts);
  // A new sequence with the tokens of another, and the page that has to be copied for it ([n, 2] int32, n 0 or 1).
  std::tuple<int64_t, at::Tensor> Fork(int64_t seq);
  void Free(int64_t seq);
  // Renumbers the pages in use to 0, 1, ...; the contents of these pages have to move ([n, 2] int32, from and to; no page is
  // both).
  at::Tensor Compact();
  int64_t Length(int64_t seq) const { return At(seq).length; }
  std::vector<int64_t> Pages(int64_t seq) const;
  int64_t FreePages() const { return static_cast<int64_t>(free_.size()); }
  int64_t NumSequences() const { return static_cast<int64_t>(sequences_.size()); }
  int64_t PageSize() const { return page_size_; }
  // [seqs, width] int32 on the CPU, -1 behind a sequence's pages; width 0: as wide as the longest needs (at least 1).
  at::Tensor Table(std::vector<int64_t> seqs, int64_t width) const;
  // [seqs] int32 on the CPU.
  at::Tensor Lengths(std::vector<int64_t> seqs) const;

 private:
  struct Sequence {
    int64_t length = 0;
    std::vector<int> pages;
  };
  const Sequence& At(int64_t seq) const;
  int64_t PagesFor(int64_t length) const { return (length + page_size_ - 1) / page_size_; }
  int Take();
  void Give(int page);
  int64_t page_size_, next_ = 0;
  std::vector<int> free_;   // the last one is taken first
  std::vector<int> users_;  // sequences that hold a page
  std::map<int64_t, Sequence> sequences_;
};

}  // namespace fo
