"""A kernel launch that fails is reported by the library call that made it, and nothing that reads what it
should have written is launched behind it.  No GPU: the calls run against a stand-in for the HIP runtime
that records launches and lets a chosen one fail (its last error stays until it is asked for)."""
import ctypes
import json
import shutil
import subprocess
import sys

import pytest

from mxtrain.ops import _lib

pytestmark = pytest.mark.usefixtures("kernel_library")

FAKE = r"""
#include <stddef.h>
#include <string.h>
typedef struct { unsigned x, y, z; } dim3_;
static dim3_ grid_, block_;
static size_t shmem_;
static void* stream_;
static int fail_at = -1, launches, last;
static unsigned long long threads;
void fake_reset(int at) { fail_at = at; launches = 0; last = 0; threads = 0; }
int fake_launches(void) { return launches; }
unsigned long long fake_threads(void) { return threads; }
void** __hipRegisterFatBinary(const void* data) { static void* h; (void)data; return &h; }
void __hipUnregisterFatBinary(void** m) { (void)m; }
void __hipRegisterFunction(void** m, const void* f, char* d, const char* n, unsigned t, void* a, void* b, void* c,
                           void* e, int* w) {}
int __hipPushCallConfiguration(dim3_ g, dim3_ b, size_t s, void* st) {
  grid_ = g; block_ = b; shmem_ = s; stream_ = st; return 0;
}
int __hipPopCallConfiguration(dim3_* g, dim3_* b, size_t* s, void** st) {
  *g = grid_; *b = block_; *s = shmem_; *st = stream_; return 0;
}
int hipLaunchKernel(const void* f, dim3_ g, dim3_ b, void** args, size_t s, void* st) {
  unsigned long long n = (unsigned long long)g.x * b.x;   /* one dimension of a launch, in threads */
  if (n > threads) threads = n;
  if (launches++ == fail_at) last = 719;
  return last;
}
int hipGetLastError(void) { int e = last; last = 0; return e; }
"""

RUN = r"""
import ctypes, json, sys
fake = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
lib = ctypes.CDLL(sys.argv[2])
fake.fake_threads.restype = ctypes.c_uint64
types = {"P": ctypes.c_void_p, "I": ctypes.c_int, "L": ctypes.c_int64, "F": ctypes.c_float}
name, sig, args = json.loads(sys.argv[3])
f = getattr(lib, name)
f.argtypes = [types[c] for c in sig]
res, n = [], 0
while not res or len(res) <= res[0][1]:
    fake.fake_reset(len(res) - 1)
    res.append((f(*args), fake.fake_launches(), fake.fake_threads()))
print(json.dumps(res))
"""


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    cc = shutil.which("cc") or shutil.which("gcc")
    if cc is None:
        pytest.skip("no C compiler")
    d = tmp_path_factory.mktemp("fake")
    (d / "fake.c").write_text(FAKE)
    subprocess.run([cc, "-shared", "-fPIC", "-w", "-o", str(d / "fake.so"), str(d / "fake.c")], check=True)
    (d / "run.py").write_text(RUN)
    return d


def _launches(fake, name, *args):
    """[(result, launches, most threads of a launch)] of the call with no launch failing, then with each in turn."""
    codes = {ctypes.c_void_p: "P", ctypes.c_int: "I", ctypes.c_int64: "L", ctypes.c_float: "F"}
    sig = "".join(codes[t] for t in _lib.SIGNATURES[name])
    out = subprocess.run([sys.executable, str(fake / "run.py"), str(fake / "fake.so"), _lib.LIB_PATH,
                          json.dumps([name, sig, args])], check=True, capture_output=True, text=True, timeout=60)
    return [tuple(r) for r in json.loads(out.stdout)]


A = 1 << 20     # some aligned address: nothing is run


def _packed_bwd(T, Hq, Hkv, D):
    floats = _lib.query64("mx_packed_attn_bwd_floats", T, Hq, Hkv, D)
    wide, narrow = Hq * D, Hkv * D
    return (A, A, A, wide, narrow, narrow, A, wide, A, wide, A, A, A, wide, A, A, narrow, narrow, A, A, A, A, T, Hq,
            Hkv, D, 0.125, 1, A, floats, None)


@pytest.mark.parametrize("T,Hq,Hkv,D,launches", [(4096, 16, 16, 64, 2), (700, 8, 1, 64, 3), (8192, 16, 16, 128, 2),
                                                 (700, 8, 1, 128, 3), (8001, 32, 8, 128, 3)])
def test_packed_attention_backward(fake, T, Hq, Hkv, D, launches):
    ok, *failed = _launches(fake, "mx_packed_attn_bwd", *_packed_bwd(T, Hq, Hkv, D))
    assert ok[:2] == (0, launches) and len(failed) == launches
    for k, (err, n, _) in enumerate(failed):
        assert err != 0 and n == k + 1, (k, failed)


@pytest.mark.parametrize("T,V,launches", [(31, 50, 2), (4096, 50304, 3), (40000, 50304, 6)])
def test_embedding_gradient(fake, T, V, launches):
    """Sums over unsorted (unwritten) token numbers would read anywhere."""
    H, words = 64, _lib.query64("mx_embedding_bwd_words", T, V, 64)
    ok, *failed = _launches(fake, "mx_embedding_bwd", A, 0, A, H, A, T, V, H, 1.0, 0, A, words, None)
    assert ok[:2] == (0, launches) and len(failed) == launches
    for k, (err, n, _) in enumerate(failed):
        assert err != 0 and n == k + 1, (k, failed)


def test_row_table(fake):
    ok, *failed = _launches(fake, "mx_packed_plan", A, 1, 3, 1000, A, A, A, A, A, None)
    assert ok[:2] == (0, 2) and [r[:2] for r in failed] == [(719, 1), (719, 2)]


@pytest.mark.parametrize("T", [16, 1003])
def test_gated_forward(fake, T):
    ok, *failed = _launches(fake, "mx_gated_fwd", A, 768, A, 768, A, A, A, A, 2048, A, A, T, 768, 2048, 768, 0, 2, 2, 4, A,
                            None)
    assert ok[0] == 0 and len(failed) == ok[1] == (2 if T == 16 else 3)
    for k, (err, n, _) in enumerate(failed):
        assert err != 0 and n == k + 1, (k, failed)


def test_gated_input_gradient(fake):
    ok, *failed = _launches(fake, "mx_gated_dx", A, A, 768, A, 1003, 768, 4096, 2, 4, A, None)
    assert ok[:2] == (0, 2) and [r[:2] for r in failed] == [(719, 1), (719, 2)]


@pytest.mark.parametrize("T", [1, 1000, (1 << 26) - 3, 1 << 26, 1 << 30])
def test_threads_of_a_lookup(fake, T):
    """A launch has fewer than 2^32 threads."""
    (ok, *_) = _launches(fake, "mx_embedding_fwd", A, A, 0, 1000, 1.0, None, None, 0, A, T, 8, None)
    assert ok[:2] == (0, 1) and 64 * min(T, 1 << 25) <= ok[2] < 1 << 32


@pytest.mark.parametrize("T,V,H", [(1 << 20, 1 << 29, 8), (1 << 29, 1 << 29, 512), (1 << 30, 1000, 8), (1 << 30, 1 << 29, 8),
                                   (1 << 30, (1 << 30) - 1, 8), (1 << 30, 1000, 1024)])
def test_threads_of_an_embedding_gradient(fake, T, V, H):
    words = _lib.query64("mx_embedding_bwd_words", T, V, H)
    (ok, *_) = _launches(fake, "mx_embedding_bwd", A, 0, A, H, A, T, V, H, 1.0, 0, A, words, None)
    if words < 0:
        assert ok[:2] == (1, 0)
    else:
        assert ok[0] == 0 and ok[2] < 1 << 32
