// raise_limit.h -- a per-kernel limit that host threads raise and none lowers (no CUDA types).
#pragma once
#include <atomic>
#include <mutex>

namespace msgl {
// Brings a limit to at least `want` by set(want), which returns 0 on success; `done` is the largest value
// set so far. Set and record happen under one lock: a thread that needs less can otherwise pass the check,
// be overtaken by one that sets and records more, and then lower what the record goes on to promise.
// The check that every later call makes is a lock-free load.
template <typename Set>
auto raise_limit(std::atomic<int>& done, int want, Set&& set) -> decltype(set(want)) {
    if (done.load(std::memory_order_acquire) >= want) return {};
    static std::mutex lock;
    std::lock_guard<std::mutex> hold(lock);
    if (done.load(std::memory_order_relaxed) >= want) return {};
    const auto e = set(want);
    if (!static_cast<int>(e)) done.store(want, std::memory_order_release);
    return e;
}
}  // namespace msgl
