// l3_errtext.h -- the text of the last error on a context.  Plain C++ (the CPU test-suite compiles it too, l3_token_hosttest.cpp).
#pragma once
#include <stdint.h>

#include <atomic>
#include <mutex>
#include <set>
#include <string>

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
    // This thread's texts, one for each of the last kMine contexts that it has one of.  Without a destructor: a thread's (and the
    // program's) last calls may come from the destructors of others.
    static constexpr uint32_t kMine = 64;
    struct Mine { uint64_t id; const char* text; };
    struct AllMine { Mine of[kMine]; uint32_t next; };
    static AllMine& mine() {
        thread_local AllMine all;         // (zeros: no context has the id 0)
        return all;
    }
    Mine* find_mine() const {
        for (Mine& m : mine().of) if (m.id == id_) return &m;
        return nullptr;
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
        Mine* m = find_mine();
        if (!m) m = &mine().of[mine().next++ % kMine];
        *m = {id_, text};
    }
    void forget_this_threads() noexcept {
        if (Mine* m = find_mine()) m->id = 0;
    }
    // of the calls that hold the context's lock
    const char* shared() const { return now_.load(std::memory_order_acquire); }
    // the calling thread's own text, if it has one that is newer
    const char* c_str() const {
        const Mine* m = find_mine();
        return m ? m->text : shared();
    }
};

}  // namespace l3
