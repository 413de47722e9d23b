"""The vote of the attention kernels over key ranges on a second walk (csrc/attn_range.hip), run on host threads: one thread per
wave of a workgroup, the source's own functions, and barriers that some waves leave late."""
import os
import re
import subprocess

import pytest

SRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lbm_amd", "csrc", "attn_range.hip")

HARNESS = r"""
#include <pthread.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <unistd.h>
#define __device__
#define __forceinline__
struct int2 { int x, y; };
static thread_local struct { int x; } threadIdx;      // the first lane of each wave
static pthread_barrier_t bar;
static int slow;
static void __syncthreads() {
  pthread_barrier_wait(&bar);
  if (threadIdx.x / 64 == slow) usleep(30000);
}
static int wave_min_i(int v) { return v; }
static int wave_max_i(int v) { return v; }
#define __builtin_amdgcn_readfirstlane(x) (x)
#define __builtin_amdgcn_ballot_w64(x) ((uint64_t)(x))
static int min(int a, int b) { return a < b ? a : b; }
static int max(int a, int b) { return a > b ? a : b; }
%s
static int sm[16], voter;
static void* wave_main(void* p) {
  const int wave = (int)(intptr_t)p;
  threadIdx.x = 64 * wave;
  const int2 range = {0, 10};
  walk_of(range, true, wave, sm);
  const bool again = any_wave(wave == voter, wave, sm);
  if (again) walk_of(range, true, wave, sm);           // the second walk starts at once
  return (void*)(intptr_t)again;
}
int main(int, char** argv) {
  voter = atoi(argv[1]);
  slow = atoi(argv[2]);
  pthread_barrier_init(&bar, 0, 4);
  pthread_t t[4];
  for (intptr_t w = 0; w < 4; ++w) pthread_create(&t[w], 0, wave_main, (void*)w);
  int got[4] = {-1, -1, -1, -1};                         // a wave that was left waiting ends the test, not the run: ten seconds
  for (int i = 0, done = 0; i < 1000 && done < 4; ++i) {
    usleep(10000);
    for (int w = 0; w < 4; ++w) {
      void* r = 0;
      if (got[w] < 0 && pthread_tryjoin_np(t[w], &r) == 0) {
        got[w] = (int)(intptr_t)r;
        ++done;
      }
    }
  }
  for (int w = 0; w < 4; ++w) printf("%%d ", got[w]);
  fflush(stdout);
  _exit(0);
}
"""


def function(text, name):
    """from the line that declares `name` (a function or a struct) to its closing brace"""
    at = re.search(rf"^[^\n/]*\b{name}\b[^\n;]*\{{$", text, re.M).start()
    return text[at:text.index("\n}", at)] + "\n};"


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    text = open(SRC).read()
    d = tmp_path_factory.mktemp("vote")
    (d / "vote.cpp").write_text(HARNESS % "\n".join(function(text, n) for n in ("struct Walk", "Walk walk_of", "bool any_wave")))
    subprocess.run(["g++", "-O1", "-pthread", "-w", str(d / "vote.cpp"), "-o", str(d / "vote")], check=True)
    return str(d / "vote")


@pytest.mark.parametrize("voter,slow", [(0, 3), (1, 0), (3, 1)])
def test_every_wave_learns_the_vote_whatever_the_others_do_next(program, voter, slow):
    out = subprocess.run([program, str(voter), str(slow)], check=True, capture_output=True, text=True).stdout.split()
    assert out == ["1"] * 4
