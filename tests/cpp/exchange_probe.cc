// leave_exchange with a thread for each CTA and one for each copy.  A copy lands some time after it was issued; it
// may not find its sender or its receiver gone.
#include <atomic>
#include <chrono>
#include <condition_variable>
#include <memory>
#include <mutex>
#include <thread>
#include <vector>

#include "../../cpu_ops_b200/csrc/exchange.h"

namespace {

using Clock = std::chrono::steady_clock;

struct Barrier {
  std::mutex m;
  std::condition_variable cv;
  int count, waiting = 0, turn = 0;
  explicit Barrier(int n) : count(n) {}
  void wait() {
    std::unique_lock<std::mutex> lock(m);
    const int mine = turn;
    if (++waiting == count) {
      waiting = 0;
      ++turn;
      cv.notify_all();
    } else {
      cv.wait(lock, [&] { return turn != mine; });
    }
  }
};

struct Cta {
  std::atomic<int> here{0};  // copies that have landed
  std::atomic<bool> late{false}, left{false};
};

struct Side {
  std::vector<std::unique_ptr<Cta>>& ctas;
  Barrier& all;
  int me;
  int* barriers;
  void tell_late() {
    for (auto& c : ctas) c->late = true;
  }
  void barrier() {
    ++*barriers;
    all.wait();
  }
  bool any_late() { return ctas[me]->late; }
  void wait_for_copies() {
    while (ctas[me]->here < static_cast<int>(ctas.size())) std::this_thread::sleep_for(std::chrono::microseconds(50));
  }
};

}  // namespace

// n CTAs; CTA i sends `delays_ms[i]` after the start, copies fly for `flight_ms`, receivers wait for `limit_ms`.
// -> copies that found a CTA gone; *late: CTAs whose first wait ran out; *barriers: barriers of one CTA.
extern "C" int probe_exchange(int n, const int* delays_ms, int flight_ms, int limit_ms, int* late, int* barriers) {
  std::vector<std::unique_ptr<Cta>> ctas;
  for (int i = 0; i < n; ++i) ctas.push_back(std::make_unique<Cta>());
  Barrier all(n);
  std::atomic<int> wrong{0}, ran_out{0};
  std::mutex m;
  std::vector<std::thread> threads, copies;
  std::vector<int> passed(n, 0);
  for (int i = 0; i < n; ++i) {
    threads.emplace_back([&, i] {
      std::this_thread::sleep_for(std::chrono::milliseconds(delays_ms[i]));
      for (int to = 0; to < n; ++to) {
        std::lock_guard<std::mutex> lock(m);
        copies.emplace_back([&, i, to] {
          std::this_thread::sleep_for(std::chrono::milliseconds(flight_ms));
          if (ctas[i]->left || ctas[to]->left) ++wrong;
          ++ctas[to]->here;
        });
      }
      const auto end = Clock::now() + std::chrono::milliseconds(limit_ms);
      while (ctas[i]->here < n && Clock::now() < end) std::this_thread::sleep_for(std::chrono::microseconds(50));
      const bool received = ctas[i]->here == n;
      if (!received) ++ran_out;
      Side side{ctas, all, i, &passed[i]};
      b200::leave_exchange(side, received);
      ctas[i]->left = true;
    });
  }
  for (auto& t : threads) t.join();
  for (auto& t : copies) t.join();
  *late = ran_out;
  *barriers = passed[0];
  return wrong;
}
