// The status text of the C ABI, shared by the library's sources.
#pragma once
#include <string>

// Sets the calling thread's fp64emu_last_error() text and returns `code`.
__attribute__((visibility("hidden"))) int fp64emu_fail(int code, const std::string& msg);
