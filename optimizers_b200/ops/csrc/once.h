// Work that is done once per key, and recorded when it has succeeded: after a call that threw, the next one does it again.
#pragma once

#include <mutex>
#include <set>

namespace ob200 {

template <typename Key>
class Once {
 public:
  template <typename Work>
  void operator()(const Key& key, Work&& work) {
    std::lock_guard<std::mutex> lock(mutex_);
    if (done_.count(key) != 0) return;
    work();
    done_.insert(key);
  }

 private:
  std::mutex mutex_;
  std::set<Key> done_;
};

}  // namespace ob200
