// How a C entry point reports: the calling thread's message (kg_last_error), and a guard that turns every C++ exception
// into it.
#pragma once
#include <exception>
#include <stdexcept>
#include <string>

namespace kgx {

int set_last_error(const std::string& msg);  // returns 1 (kgx_api.cpp)

template <typename F>
int guarded(F&& f) {
  try {
    f();
    return 0;
  } catch (const std::exception& e) {
    return set_last_error(e.what());
  } catch (...) {
    return set_last_error("unknown error");
  }
}

}  // namespace kgx
