"""xpu_pages_* when host memory runs out, in any allocation of a call: an error
code and no C++ exception at the C entry, and the pages as they were. The
sources are built here with an operator new that fails on demand."""
import os
import shutil
import subprocess

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include "xpu_playground_amd/csrc/pages.cpp"
#include <cstdio>
#include <cstdlib>
#include <new>

static long fail_at = -1;  // the allocation that fails, and all behind it
static long allocations = 0;
void *operator new(std::size_t n) {
  if (fail_at >= 0 && allocations++ >= fail_at) throw std::bad_alloc();
  if (void *p = std::malloc(n)) return p;
  throw std::bad_alloc();
}
void operator delete(void *p) noexcept { std::free(p); }
void operator delete(void *p, std::size_t) noexcept { std::free(p); }
namespace xpu {
std::string last;
int set_error(int code, const std::string &message) { last = message; return code; }
}

static uint32_t held(xpu_pages *p) {
  uint32_t sum = 0, n = 0;
  for (uint32_t i = 0; i < 8; ++i) { xpu_pages_holders(p, i, &n); sum = sum * 5 + n; }
  xpu_pages_free_count(p, &n);
  return sum * 9 + n;
}

template <typename Call> static int check(const char *name, bool succeeds, Call &&call) {
  int bad = 0;
  for (long k = 0; k < 40; ++k) {
    xpu_pages *p = nullptr;
    uint32_t ids[8] = {};
    if (xpu_pages_create(8, &p) || xpu_pages_take(p, 5, ids) || xpu_pages_share(p, ids, 2) || xpu_pages_release(p, ids + 2, 1)) return 1;
    const uint32_t before = held(p);
    xpu::last = std::string();
    int rc = -1;
    fail_at = k, allocations = 0;
    try { rc = call(p); } catch (...) { rc = -2; }
    const bool ran_out = allocations > k;
    fail_at = -1;
    if (rc == -2) std::printf("%s: an exception left it (allocation %ld)\n", name, k), ++bad;
    else if (ran_out && rc == 0) std::printf("%s: 0 without memory (allocation %ld)\n", name, k), ++bad;
    else if (!ran_out && (rc == 0) != succeeds) std::printf("%s: %d\n", name, rc), ++bad;
    if (rc != 0 && held(p) != before) std::printf("%s: changed the pages (allocation %ld)\n", name, k), ++bad;
    xpu_pages_destroy(p);
    if (!ran_out) return bad;
  }
  return bad + 1;
}

int main() {
  int bad = 0;
  uint32_t n = 0, ids[8], src[8], dst[8];
  bad += check("create", true, [&](xpu_pages *) { xpu_pages *q = nullptr; int rc = xpu_pages_create(8, &q); if (!rc) xpu_pages_destroy(q); return rc; });
  bad += check("create null", false, [&](xpu_pages *) { return xpu_pages_create(8, nullptr); });
  bad += check("create none", false, [&](xpu_pages *) { xpu_pages *q; return xpu_pages_create(0, &q); });
  bad += check("free_count null", false, [&](xpu_pages *p) { return xpu_pages_free_count(p, nullptr); });
  bad += check("holders null", false, [&](xpu_pages *) { return xpu_pages_holders(nullptr, 0, &n); });
  bad += check("holders none", false, [&](xpu_pages *p) { return xpu_pages_holders(p, 8, &n); });
  bad += check("take", true, [&](xpu_pages *p) { return xpu_pages_take(p, 3, ids); });
  bad += check("take many", false, [&](xpu_pages *p) { return xpu_pages_take(p, 9, ids); });
  bad += check("share", true, [&](xpu_pages *p) { uint32_t a[] = {0, 3, 4}; return xpu_pages_share(p, a, 3); });
  bad += check("share free", false, [&](xpu_pages *p) { uint32_t a[] = {0, 2}; return xpu_pages_share(p, a, 2); });
  bad += check("release", true, [&](xpu_pages *p) { uint32_t a[] = {0, 3, 4, 0}; return xpu_pages_release(p, a, 4); });
  bad += check("release often", false, [&](xpu_pages *p) { uint32_t a[] = {3, 4, 3}; return xpu_pages_release(p, a, 3); });
  bad += check("own", true, [&](xpu_pages *p) { uint32_t a[] = {0, 3, 1}; return xpu_pages_own(p, a, 3, src, dst, &n); });
  bad += check("own twice", false, [&](xpu_pages *p) { uint32_t a[] = {0, 0}; return xpu_pages_own(p, a, 2, src, dst, &n); });
  bad += check("compact", true, [&](xpu_pages *p) { return xpu_pages_compact(p, src, dst, &n); });
  bad += check("compact null", false, [&](xpu_pages *p) { return xpu_pages_compact(p, src, nullptr, &n); });
  bad += check("renumber", true, [&](xpu_pages *) { uint32_t a[] = {4, 1}, s[] = {4}, d[] = {2}; return xpu_pages_renumber(s, d, 1, a, 2); });
  bad += check("renumber null", false, [&](xpu_pages *) { return xpu_pages_renumber(nullptr, dst, 1, nullptr, 0); });
  if (!bad) std::puts("fine");
  return bad != 0;
}
"""


@pytest.mark.skipif(not shutil.which("g++"), reason="no host compiler")
def test_every_allocation_may_fail(tmp_path):
    source, program = tmp_path / "main.cpp", tmp_path / "main"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", "-I", REPO, "-I",
                    os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "include"), str(source), "-o", str(program)],
                   check=True)
    run = subprocess.run([str(program)], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and run.stdout == "fine\n", run.stdout + run.stderr
