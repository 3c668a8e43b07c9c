// known.h -- answers of the device that depend on a key alone, asked for once.
#pragma once

#include <map>
#include <mutex>
#include <new>

namespace det {

// get() gives what ask(&value) gave for the key.  Only an answer is kept: a
// query that fails hands its error on, and the next call asks again; so it does
// where there is no memory to keep the answer.
template <typename Key, typename Value>
class Known {
 public:
  template <typename Ask>
  auto get(const Key& key, Value* out, Ask ask) -> decltype(ask(out)) {
    std::lock_guard<std::mutex> lock(mu_);
    const auto it = known_.find(key);
    if (it != known_.end()) {
      *out = it->second;
      return {};
    }
    Value v{};
    const auto error = ask(&v);
    if (error != decltype(ask(out)){}) return error;
    *out = v;
    try {
      known_.emplace(key, v);
    } catch (const std::bad_alloc&) {
    }
    return error;
  }

 private:
  std::mutex mu_;
  std::map<Key, Value> known_;
};

}  // namespace det
