// Host bookkeeping of a paged key-value cache: which pages a sequence owns, how many sequences
// share a page, and which pages are free.  Plain C++ (no CUDA): the device side is the page copies
// that fork and compact ask for.  moe-680m keeps one contiguous cache region per layer and one
// sequence (src/memory.rs:61-85); sequences that share pages have no counterpart there.
//
// Invariants between calls: a page with users > 0 is in the table of exactly `users` sequences; a
// partly filled page (only ever a sequence's last) has one user, so appending never writes into a
// shared page; pages are handed out lowest free id first.  Every call checks all of its arguments
// first and then either does all of its work or, with an error, none.
#pragma once
#include <cstdint>
#include <functional>
#include <numeric>
#include <queue>
#include <string>
#include <utility>
#include <vector>

#include "../../include/moe_b200.h"

namespace moe {

class KvPages {
public:
    using Moves = std::vector<std::pair<uint32_t, uint32_t>>;  // (from, to) pages
    using Copy = std::function<int(const Moves&)>;             // makes the copies on the device: MOE_OK or an error

    KvPages(uint32_t n_pages, uint32_t page_size) : page_size_(page_size), users_(n_pages, 0) {
        std::vector<uint32_t> all(n_pages);
        std::iota(all.begin(), all.end(), 0u);
        free_ = Heap(std::greater<uint32_t>(), std::move(all));
    }

    uint32_t n_pages() const { return static_cast<uint32_t>(users_.size()); }
    uint32_t n_free() const { return static_cast<uint32_t>(free_.size()); }

    // n new empty sequences.  A handle is (generation << 32 | slot + 1), never 0; the generation
    // tells a freed sequence's handle from its slot's next owner.
    int create(uint32_t n, uint64_t* out, std::string* err) {
        if (seqs_.size() - idle_.size() + n > kMaxSeqs) return fail(err, MOE_E_UNSUPPORTED, "more than 1048576 sequences");
        const size_t reuse = idle_.size() < n ? idle_.size() : n;
        seqs_.reserve(seqs_.size() + (n - reuse));
        idle_.reserve(seqs_.size() + (n - reuse));  // freeing never allocates
        for (uint32_t i = 0; i < n; ++i) {
            uint32_t slot;
            if (!idle_.empty()) {
                slot = idle_.back();
                idle_.pop_back();
            } else {
                slot = static_cast<uint32_t>(seqs_.size());
                seqs_.emplace_back();
            }
            seqs_[slot].live = true;
            out[i] = handle(slot);
        }
        return MOE_OK;
    }

    // Room for add[i] more tokens in each sequence.
    int extend(const uint64_t* h, uint32_t n, const uint64_t* add, std::string* err) {
        int rc = check(h, n, false, err);
        if (rc) return rc;
        uint64_t need = 0;
        for (uint32_t i = 0; i < n; ++i) {
            Seq& s = at(h[i]);
            if (add[i] > kMaxTokens || s.len + add[i] > kMaxTokens)
                return fail(err, MOE_E_UNSUPPORTED, "a sequence longer than 2147483392 tokens");
            need += pages_of(s.len + add[i]) - s.pages.size();
        }
        if (need > free_.size()) return fail(err, MOE_E_OOM, "cache pages: need " + std::to_string(need) + ", " + std::to_string(free_.size()) + " free");
        for (uint32_t i = 0; i < n; ++i) at(h[i]).pages.reserve(pages_of(at(h[i]).len + add[i]));
        for (uint32_t i = 0; i < n; ++i) {
            Seq& s = at(h[i]);
            s.len += add[i];
            while (s.pages.size() < pages_of(s.len)) s.pages.push_back(take());
        }
        return MOE_OK;
    }

    // One child per parent (a parent may be given more than once): full pages are shared, a partly
    // filled last page gets a page of its own, listed in `copies` and copied by `copy`.
    int fork(const uint64_t* parents, uint32_t n, uint64_t* children, Moves* copies, std::string* err, const Copy& copy = nullptr) {
        int rc = check(parents, n, true, err);
        if (rc) return rc;
        uint64_t need = 0;
        for (uint32_t i = 0; i < n; ++i) need += at(parents[i]).len % page_size_ != 0;
        if (need > free_.size()) return fail(err, MOE_E_OOM, "cache pages: need " + std::to_string(need) + ", " + std::to_string(free_.size()) + " free");
        std::vector<std::vector<uint32_t>> tables(n);
        for (uint32_t i = 0; i < n; ++i) tables[i] = at(parents[i]).pages;
        copies->reserve(need);
        std::vector<uint64_t> made(n);
        if ((rc = create(n, made.data(), err))) return rc;
        for (uint32_t i = 0; i < n; ++i) {
            Seq& child = at(made[i]);
            child.len = at(parents[i]).len;
            child.pages.swap(tables[i]);
            const bool part = child.len % page_size_ != 0;
            for (size_t j = 0; j + (part ? 1 : 0) < child.pages.size(); ++j) ++users_[child.pages[j]];
            if (part) {
                const uint32_t p = take();
                copies->emplace_back(child.pages.back(), p);
                child.pages.back() = p;
            }
        }
        if (copy) {
            try {
                rc = copy(*copies);
            } catch (...) {
                free(made.data(), n, err);
                throw;
            }
            if (rc) {
                free(made.data(), n, err);  // of living sequences, each once: it cannot fail
                return rc;
            }
        }
        for (uint32_t i = 0; i < n; ++i) children[i] = made[i];
        return MOE_OK;
    }

    int free(const uint64_t* h, uint32_t n, std::string* err) {
        int rc = check(h, n, false, err);
        if (rc) return rc;
        for (uint32_t i = 0; i < n; ++i) {
            Seq& s = at(h[i]);
            for (uint32_t p : s.pages)
                if (--users_[p] == 0) free_.push(p);  // within the heap's first size: no allocation
            s.pages.clear();
            s.len = 0;
            s.live = false;
            ++s.gen;
            idle_.push_back(slot_of(h[i]));
        }
        return MOE_OK;
    }

    // Moves the used pages into ids [0, used): the i-th used page at or above that bound goes to the
    // i-th free page below it, so no page is both read and written.  The copies are made (`copy`) before anything changes:
    // they write free pages only.
    int compact(Moves* moves, const Copy& copy = nullptr) {
        const uint32_t used = n_pages() - n_free();
        std::vector<uint32_t> to(users_.size()), rest;
        for (uint32_t p = 0; p < to.size(); ++p) to[p] = p;
        moves->reserve(used);
        rest.reserve(users_.size());  // the heap never grows past it
        uint32_t hole = 0;
        for (uint32_t p = used; p < users_.size(); ++p) {
            rest.push_back(p);
            if (users_[p] == 0) continue;
            while (users_[hole] != 0) ++hole;
            moves->emplace_back(p, hole);
            to[p] = hole++;
        }
        if (copy)
            if (const int rc = copy(*moves)) return rc;
        for (const auto& m : *moves) std::swap(users_[m.first], users_[m.second]);
        for (Seq& s : seqs_)
            for (uint32_t& p : s.pages) p = to[p];
        free_ = Heap(std::greater<uint32_t>(), std::move(rest));
        return MOE_OK;
    }

    // The table rows of n sequences ([n][max_pages], unused entries 0), then their n lengths.
    int tables(const uint64_t* h, uint32_t n, uint32_t max_pages, std::vector<int32_t>* out, std::string* err) {
        int rc = check(h, n, true, err);
        if (rc) return rc;
        out->assign(static_cast<size_t>(n) * max_pages + n, 0);
        for (uint32_t i = 0; i < n; ++i) {
            const Seq& s = at(h[i]);
            if (s.pages.size() > max_pages)
                return fail(err, MOE_E_INVALID, "sequence " + std::to_string(i) + " has " + std::to_string(s.pages.size()) +
                                                    " pages, the table rows " + std::to_string(max_pages));
            for (size_t j = 0; j < s.pages.size(); ++j) (*out)[static_cast<size_t>(i) * max_pages + j] = static_cast<int32_t>(s.pages[j]);
            (*out)[static_cast<size_t>(n) * max_pages + i] = static_cast<int32_t>(s.len);
        }
        return MOE_OK;
    }

    // Page copies given by a caller: ids in range, no page written twice, none both read and written.
    int check_copies(const uint64_t* src, const uint64_t* dst, uint32_t n, std::string* err) const {
        std::vector<uint8_t> written(users_.size(), 0);
        for (uint32_t i = 0; i < n; ++i) {
            if (src[i] >= users_.size() || dst[i] >= users_.size())
                return fail(err, MOE_E_INVALID, "copy " + std::to_string(i) + ": page outside the cache's " + std::to_string(users_.size()));
            if (written[dst[i]]) return fail(err, MOE_E_INVALID, "copy " + std::to_string(i) + ": page " + std::to_string(dst[i]) + " written twice");
            written[dst[i]] = 1;
        }
        for (uint32_t i = 0; i < n; ++i)
            if (written[src[i]]) return fail(err, MOE_E_INVALID, "copy " + std::to_string(i) + ": page " + std::to_string(src[i]) + " is read and written");
        return MOE_OK;
    }

private:
    static constexpr uint64_t kMaxTokens = 2147483392ull;  // a length and a tile behind it fit 32 bits
    static constexpr size_t kMaxSeqs = 1u << 20;
    using Heap = std::priority_queue<uint32_t, std::vector<uint32_t>, std::greater<uint32_t>>;
    struct Seq {
        uint32_t gen = 0;
        bool live = false;
        uint64_t len = 0;
        std::vector<uint32_t> pages;
        uint64_t seen = 0;  // the last check() that met it
    };

    static int fail(std::string* err, int code, const std::string& what) {
        *err = what;
        return code;
    }
    static uint32_t slot_of(uint64_t h) { return static_cast<uint32_t>(h & 0xFFFFFFFFu) - 1; }
    uint64_t handle(uint32_t slot) const { return static_cast<uint64_t>(seqs_[slot].gen) << 32 | (slot + 1); }
    Seq& at(uint64_t h) { return seqs_[slot_of(h)]; }
    uint64_t pages_of(uint64_t len) const { return (len + page_size_ - 1) / page_size_; }
    uint32_t take() {
        const uint32_t p = free_.top();
        free_.pop();
        users_[p] = 1;
        return p;
    }
    int check(const uint64_t* h, uint32_t n, bool repeats, std::string* err) {
        ++checks_;
        for (uint32_t i = 0; i < n; ++i) {
            const uint64_t low = h[i] & 0xFFFFFFFFu;
            if (low == 0 || low > seqs_.size() || !at(h[i]).live || at(h[i]).gen != h[i] >> 32)
                return fail(err, MOE_E_INVALID, "sequence handle " + std::to_string(i) + " is not of a living sequence");
            if (!repeats && at(h[i]).seen == checks_) return fail(err, MOE_E_INVALID, "sequence handle " + std::to_string(i) + " given twice");
            at(h[i]).seen = checks_;
        }
        return MOE_OK;
    }

    uint32_t page_size_;
    std::vector<uint32_t> users_;
    Heap free_;
    std::vector<Seq> seqs_;
    std::vector<uint32_t> idle_;
    uint64_t checks_ = 0;
};

}  // namespace moe
