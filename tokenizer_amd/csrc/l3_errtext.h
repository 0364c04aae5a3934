// l3_errtext.h -- the text of the last error on a context.  Plain C++ (the CPU test-suite compiles it too, l3_token_hosttest.cpp).
#pragma once
#include <stdint.h>

#include <atomic>
#include <mutex>
#include <set>
#include <string>
#include <utility>
#include <vector>

namespace l3 {

// Calls that hold the context's lock assign to it; calls that take no lock, and may run at the same time, leave their text for the
// thread that made them.  Whoever asks does so without a lock while another call may fail, so no text is ever changed or freed
// before the context is: each different one is kept once (there are a few dozen messages), and what changes is a pointer.
class ErrText {
    const uint64_t id_ = next_id();       // (an address may be a later context's, too)
    std::mutex mu_;                       // held for the length of an insertion
    std::set<std::string> texts_;
    std::atomic<const char*> now_{""};

    static uint64_t next_id() {
        static std::atomic<uint64_t> n{0};
        return ++n;
    }
    typedef std::pair<uint64_t, const char*> Mine;
    static std::vector<Mine>& mine() {    // this thread's texts, one for each context
        thread_local std::vector<Mine> texts;
        return texts;
    }
    const char* keep(const std::string& text) {
        std::lock_guard<std::mutex> lk(mu_);
        return texts_.insert(text).first->c_str();
    }

  public:
    ErrText& operator=(const std::string& text) {
        now_.store(keep(text), std::memory_order_release);
        forget_this_threads();
        return *this;
    }
    // `what` is a string literal: where there is no memory for the whole text, it stands alone
    void leave_for_this_thread(const char* what, const char* more) noexcept {
        const char* text = what;
        try {
            text = keep(std::string(what) + more);
        } catch (...) {
        }
        try {
            forget_this_threads();
            mine().emplace_back(id_, text);
        } catch (...) {
        }
    }
    void forget_this_threads() noexcept {
        std::vector<Mine>& m = mine();
        for (size_t i = 0; i < m.size(); i++)
            if (m[i].first == id_) { m[i] = m.back(); m.pop_back(); return; }
    }
    // of the calls that hold the context's lock
    const char* shared() const { return now_.load(std::memory_order_acquire); }
    // the calling thread's own text, if it has one that is newer
    const char* c_str() const {
        for (const Mine& m : mine()) if (m.first == id_) return m.second;
        return shared();
    }
};

}  // namespace l3
