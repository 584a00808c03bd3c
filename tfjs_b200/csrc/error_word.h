// What kernels report in the context's device error word.  A wait that gave up stores its code, below
// kBadInput, over whatever is there; inputs that only the device can check add their bits, which
// leave a code as it is.  So a wait that gave up is never hidden by a bad input.
#pragma once

enum { kBadPage = 1 << 16, kBadLength = 1 << 17, kBadInput = kBadPage };

// Code of the wait that gave up, or 0.
inline int error_word_timeout(int word) { return word & (kBadInput - 1); }

// What is wrong with the inputs, or null.
inline const char* error_word_input(int word) {
  const bool page = (word & kBadPage) != 0, length = (word & kBadLength) != 0;
  if (page && length)
    return "a kernel needed a page that its page table does not name (outside the pool); the slots of that page "
           "were left out.  A row's length is outside what its tensors hold; it was clamped";
  if (page)
    return "a kernel needed a page that its page table does not name (outside the pool); the slots of that page "
           "were left out";
  return length ? "a row's length is outside what its tensors hold; it was clamped" : nullptr;
}
