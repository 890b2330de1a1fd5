// Checks of csrc/device_count.h: prints "ok" or what went wrong.
#include <cstdio>
#include <thread>
#include <vector>

#include "device_count.h"

#define EXPECT(x)                                       \
  do {                                                  \
    if (!(x)) return std::printf("line %d: %s\n", __LINE__, #x), 1; \
  } while (0)

int main() {
  static lsc::DeviceCount count;
  int asked = 0;
  auto answers = [&](int n) { return [&asked, n](int* out) { return ++asked, *out = n, true; }; };
  auto fails = [&](int* out) { return ++asked, *out = 5, false; };
  EXPECT(count.get(0, fails) == -1 && asked == 1);
  EXPECT(count.get(0, answers(18)) == 18 && asked == 2);  // the failure was not kept
  EXPECT(count.get(0, fails) == 18 && asked == 2);        // the answer was
  EXPECT(count.get(1, answers(0)) == 0 && asked == 3);    // another device is asked itself
  EXPECT(count.get(1, answers(7)) == 0 && asked == 3);
  EXPECT(count.get(lsc::kMaxDevices - 1, fails) == -1 && asked == 4);
  EXPECT(count.get(0, answers(3)) == 18 && asked == 4);
  static lsc::DeviceCount shared;
  std::vector<std::thread> threads;
  std::atomic<int> wrong{0};
  for (int t = 0; t < 8; ++t)
    threads.emplace_back([&] {
      for (int i = 0; i < 1000; ++i)
        for (int d = 0; d < lsc::kMaxDevices; ++d)
          if (shared.get(d, [d](int* out) { return *out = d, true; }) != d) ++wrong;
    });
  for (auto& t : threads) t.join();
  EXPECT(wrong == 0);
  std::printf("ok\n");
  return 0;
}
