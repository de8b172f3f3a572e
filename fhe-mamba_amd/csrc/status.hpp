// Status codes of the C ABI: the calling thread's last message, and the
// translation of C++ exceptions into codes.  No exception crosses the ABI.
#pragma once

#include <stdexcept>
#include <string>

#include "../../include/fhecore.h"
#include "context.hpp"

namespace fhe {

inline thread_local std::string last_error;

template <typename F>
int guard(F&& f) {
  try {
    f();
    return FHE_OK;
  } catch (const ArgError& e) {
    last_error = e.what();
    return FHE_ERR_ARG;
  } catch (const HipError& e) {
    last_error = e.what();
    return FHE_ERR_HIP;
  } catch (const StateError& e) {
    last_error = e.what();
    return FHE_ERR_STATE;
  } catch (const std::out_of_range& e) {
    last_error = e.what();
    return FHE_ERR_RANGE;
  } catch (const std::exception& e) {
    last_error = e.what();
    return FHE_ERR_INTERNAL;
  } catch (...) {
    last_error = "unknown error";
    return FHE_ERR_INTERNAL;
  }
}

inline void need(bool ok, const char* msg) {
  if (!ok) throw ArgError(msg);
}

}  // namespace fhe
