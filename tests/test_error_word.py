"""The device error word: what it says about waits that gave up and about inputs, in any order of the
kernels that report."""
import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "tfjs_b200", "csrc")

PROGRAM = r"""
#include <stdio.h>
#include <string.h>
#include "error_word.h"
// a wait stores its code, an input adds its bit
static void report(int* word, int value) { value < kBadInput ? *word = value : *word |= value; }
int main() {
  const int values[] = {4, kBadPage, kBadLength, 9};
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j)
      for (int k = 0; k < 4; ++k) {
        int word = 0, waits = 0;
        const int order[] = {values[i], values[j], values[k]};
        for (int v : order) {
          report(&word, v);
          if (v < kBadInput) waits = v;
        }
        if (error_word_timeout(word) != waits) return 1;
        const char* text = error_word_input(word);
        if (waits) continue;
        bool page = false, length = false;
        for (int v : order) page |= v == kBadPage, length |= v == kBadLength;
        if (!text || (strstr(text, "page") != nullptr) != page || (strstr(text, "length") != nullptr) != length) return 2;
      }
  return error_word_timeout(0) || error_word_input(0) || error_word_input(7) ? 3 : 0;
}
"""


def test_a_wait_that_gave_up_is_never_hidden(tmp_path):
    source, program = tmp_path / "word.cc", tmp_path / "word"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-I", CSRC, str(source), "-o", str(program)], check=True)
    assert subprocess.run([str(program)]).returncode == 0


def test_kernels_report_as_the_word_is_read():
    """Inputs by atomicOr, waits by a code that is below the inputs' bits."""
    codes = 0
    for name in os.listdir(CSRC):
        if not name.endswith((".cu", ".cuh", ".h")):
            continue
        text = open(os.path.join(CSRC, name)).read()
        for value in re.findall(r"atomicExch\([\w.]*flag, ([^)]*)\)", text):
            assert 0 < int(value) < 1 << 16, (name, value)
            codes += 1
        assert not re.search(r"atomicExch\([^;]*kBad", text), name
    assert codes > 20
