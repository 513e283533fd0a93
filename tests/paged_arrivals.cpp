// The arrival counters' protocol (dooms_b200/csrc/kernels/arrivals.h) on the host: every order in which the memory operations of a few arrivers can follow one another.
#include "arrivals.h"

#include <vector>

using namespace dooms::cuda;

namespace {

struct Pause {};
// What an arriver's operations gave so far; one more is let through, and then it pauses.
struct Arriver {
    bool failed;
    std::vector<Arrivals> log;
    bool over = false;
    Arrival result = Arrival::kNotLast;
};
struct Memory {
    Arrivals * at;
    std::vector<Arrivals> * log;
    size_t * next;
    bool * let;
    template <class F> Arrivals step(F f) const {
        if (*next == log->size()) {
            if (!*let) throw Pause{};
            *let = false;
            log->push_back(f());
        }
        return (*log)[(*next)++];
    }
    Arrivals load() const { return step([&] { return *at; }); }
    Arrivals swap(Arrivals was, Arrivals to) const { return step([&] { const Arrivals v = *at; if (v == was) *at = to; return v; }); }
    Arrivals add(Arrivals n) const { return step([&] { const Arrivals v = *at; *at += n; return v; }); }
    void store(Arrivals to) const { step([&] { *at = to; return to; }); }
};

struct Search {
    Arrivals call;
    long long orders = 0, wrong = 0;
    void go(Arrivals memory, const std::vector<Arriver> & all) {
        bool more = false;
        for (size_t i = 0; i < all.size(); i++) {
            if (all[i].over) continue;
            more = true;
            std::vector<Arriver> next = all;
            Arrivals now = memory;
            size_t at = 0;
            bool let = true;
            try {
                next[i].result = arrive(Memory{&now, &next[i].log, &at, &let}, call, int(all.size()), next[i].failed);
                next[i].over = true;
            } catch (Pause) {}
            go(now, next);
        }
        if (more) return;
        orders++;
        int last = 0;
        bool failed = false, said = false;
        for (const Arriver & a : all) { last += a.result != Arrival::kNotLast; failed |= a.failed; said |= a.result == Arrival::kLastAfterFailure; }
        if (last != 1 || said != failed || memory != 0) wrong++;
    }
};

}  // namespace

// The number of orders of `n` arrivers of call `call`, those of the bits of `failed` failing, from the counter's content `start`; *wrong: of those in which not exactly one was
// the last, it did not know of a failure (or knew of one that was none), or the counter was not zero in the end.
extern "C" long long arrivals_orders(int n, unsigned long long call, unsigned failed, unsigned long long start, long long * wrong) {
    std::vector<Arriver> all;
    for (int i = 0; i < n; i++) all.push_back({(failed >> i & 1) != 0, {}});
    Search s{call};
    s.go(start, all);
    *wrong = s.wrong;
    return s.orders;
}
