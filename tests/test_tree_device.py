"""The host side of the tree and cache calls against a stand-in HIP runtime (tests/fakehip.c):
what they leave behind of the thread's current device.  Each test runs in a child process that
preloads it; nothing is computed."""
import os
import shutil
import subprocess
import sys

import pytest

from xwen_amd import _lib

HERE = os.path.dirname(os.path.abspath(__file__))

COMMON = """
import ctypes as C
from xwen_amd import _lib
lib, rt = _lib.load(), C.CDLL(None)
for f in ("fake_used", "fake_launches", "fake_work_items"):
    getattr(rt, f).restype = C.c_int64
rt.fake_room.argtypes = [C.c_int64]
P = 0x7f0000001000

def device():
    d = C.c_int(-1)
    rt.hipGetDevice(C.byref(d))
    return d.value

def kv():
    return _lib.Kv(P, P, 64 * 512, 512, 64)

def cache(dims=(4, 16, 16, 8, 64, 64), on=0):
    h = C.c_void_p()
    return lib.xs_cache_create(on, C.byref(_lib.CacheDims(*dims)), C.byref(h)), h

def calls(cache_ctx, ctx):
    a = _lib.TreeAttendArgs(dtype=_lib.BF16, head_dim=64, seqs=4, nodes=16, q_heads=16, kv_heads=8, q=P, q_seq_stride=16 * 1024,
                            q_node_stride=1024, q_head_stride=64, cache=kv(), capacity=64, len=P, fresh=kv(), parent=P, scale=0.1,
                            out=P + 4096, out_seq_stride=16 * 1024, out_node_stride=1024, out_head_stride=64, seq_status=P)
    c = _lib.CacheCommitArgs(dtype=_lib.BF16, head_dim=64, seqs=4, nodes=16, q_heads=8, kv_heads=8, cache=kv(), capacity=64, len=P,
                             fresh=kv(), path=P, path_ld=16, n_path=P, new_len=P + 64, slot_ld=64, seq_status=P)
    e = _lib.CacheEvictArgs(dtype=_lib.BF16, head_dim=64, seqs=4, kv_heads=8, cache=kv(), capacity=64, len=P, mass=P, new_mass=P, pos=P,
                            new_pos=P, slot_ld=64, next_pos=P, keep=40, sinks=4, recent=8, new_len=P + 64, seq_status=P)
    v = _lib.VerifyTreeArgs(logits=P, seqs=4, nodes=16, ld=1000, width=1000, enc=1000, params=P, uniforms=P, tokens=P, parent=P,
                            row_token=P, row_status=P, accepted=P, path=P, committed=P, n_committed=P, seq_status=P)
    return [(lib.xs_tree_attend, cache_ctx, a), (lib.xs_cache_commit, cache_ctx, c), (lib.xs_cache_evict, cache_ctx, e),
            (lib.xs_verify_tree, ctx, v)]
"""


@pytest.fixture(scope="module")
def runtime(tmp_path_factory):
    if not shutil.which("gcc"):
        pytest.skip("gcc is not installed")
    so = str(tmp_path_factory.mktemp("fakehip") / "libfakehip.so")
    subprocess.run(["gcc", "-O1", "-Wall", "-Wextra", "-shared", "-fPIC", os.path.join(HERE, "fakehip.c"), "-o", so], check=True)
    return so


def child(runtime, body):
    before = os.environ.get("LD_PRELOAD")
    env = dict(os.environ, LD_PRELOAD=f"{runtime} {before}" if before else runtime, PYTHONPATH=_lib.ROOT)
    r = subprocess.run([sys.executable, "-c", COMMON + body], cwd=_lib.ROOT, env=env, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip().endswith("done"), r.stdout + r.stderr
    return r.stdout


def test_calls_leave_the_current_device(runtime):
    child(runtime, """
rc, h = cache()
ctx = C.c_void_p()
assert rc == 0 and lib.xs_create(0, 64, 1000, 0, C.byref(ctx)) == 0
for now in (0, 1):
    rt.hipSetDevice(now)
    for call, c, args in calls(h, ctx):
        before = rt.fake_launches()
        assert call(c, C.byref(args)) == 0 and rt.fake_launches() > before, call
        assert device() == now, (call.__name__, now, device())
rt.hipSetDevice(1)
rc, other = cache()
assert rc == 0 and device() == 1
assert lib.xs_cache_destroy(other) == 0 and lib.xs_cache_destroy(h) == 0 and device() == 1
print("done")
""")


def test_a_context_that_cannot_be_made_leaves_nothing_behind(runtime):
    """Too little memory at every allocation in turn, sizes that no memory holds, a device that is
    not there: XS_ERR_HIP, no memory kept, the current device as it was, and no error that the
    thread's next HIP call would report."""
    child(runtime, """
rc, h = cache()
assert rc == 0
whole = rt.fake_used()
assert lib.xs_cache_destroy(h) == 0 and rt.fake_used() == 0
rt.hipSetDevice(1)
for room in sorted({0, 1, whole // 2, whole - 1, *range(0, whole, max(1, whole // 64))}):
    rt.fake_room(room)
    rc, h = cache()
    assert rc == _lib.XS_ERR_HIP and not h.value and rt.fake_used() == 0 and device() == 1, room
    assert rt.fake_last_error() == 0, (room, rt.fake_last_error())
rt.fake_room(1 << 40)
rc, h = cache((65536, 64, 4096, 4096, 256, 1 << 28))
assert rc == _lib.XS_ERR_HIP and not h.value and rt.fake_used() == 0 and rt.fake_last_error() == 0
rc, h = cache(on=7)
assert rc == _lib.XS_ERR_HIP and not h.value and device() == 1 and rt.fake_last_error() == 0
print("done")
""")


def test_a_context_holds_what_its_calls_can_use(runtime):
    """The partial results of split attention: for single tokens no tree's, none where no call is
    split; and every call within a context's sizes has room for its own."""
    out = child(runtime, """
import random
def size(*dims):
    rc, h = cache(dims)
    assert rc == 0
    n = rt.fake_used()
    lib.xs_cache_destroy(h)
    return n
def evict(seqs, kv, cap):  # the lists of moves and the bitmap
    return seqs * kv * ((cap + 63) // 64 * 8 + (cap // 2 + 1) * 8 + 4)
cases = {"decode": (16, 1, 32, 8, 128, 8192), "tree": (16, 64, 32, 8, 128, 8192), "one": (1, 64, 32, 8, 128, 131072),
         "short": (16, 64, 32, 8, 128, 448)}
for name, d in cases.items():
    print(name, size(*d) - evict(d[0], d[3], d[5]))
rng = random.Random(1)
for _ in range(1500):
    kv = rng.choice([1, 2, 3, 8, 16])
    dims = dict(seqs=rng.choice([1, 2, 7, 64, 900]), nodes=rng.choice([1, 2, 5, 16, 33, 64]), g=rng.choice([1, 2, 4, 7, 16]),
                dim=rng.choice([8, 64, 72, 128, 136, 256]), cap=rng.choice([1, 64, 300, 480, 512, 700, 2000, 9000, 70000, 1 << 20]))
    rc, h = cache((dims["seqs"], dims["nodes"], kv * dims["g"], kv, dims["dim"], dims["cap"]))
    assert rc == 0
    for _ in range(12):
        k = rng.randint(1, kv)
        q = k * rng.randint(1, kv * dims["g"] // k)
        seqs, nodes, cap = rng.randint(1, dims["seqs"]), rng.randint(1, dims["nodes"]), rng.randint(1, dims["cap"])
        dim = 8 * rng.randint(1, dims["dim"] // 8)
        if rng.random() < 0.5:
            k, q, seqs, nodes, cap, dim = kv, kv * dims["g"], dims["seqs"], dims["nodes"], dims["cap"], dims["dim"]
        stride = _lib.Kv(P, P, cap * k * 256, k * 256, 256)
        a = _lib.TreeAttendArgs(dtype=rng.randint(0, 1), head_dim=dim, seqs=seqs, nodes=nodes, q_heads=q, kv_heads=k, q=P,
                                q_seq_stride=nodes * q * 256, q_node_stride=q * 256, q_head_stride=256, cache=stride, capacity=cap, len=P,
                                fresh=stride, parent=P, scale=0.1, out=P + 4096, out_seq_stride=nodes * q * 256, out_node_stride=q * 256,
                                out_head_stride=256, seq_status=P)
        assert lib.xs_tree_attend(h, C.byref(a)) == 0, (dims, kv, seqs, nodes, q, k, dim, cap)
    lib.xs_cache_destroy(h)
print("done")
""")
    got = {k: int(v) for k, v in (line.split() for line in out.splitlines()[:-1])}
    assert got["short"] == 0
    # 256 CUs of 2 workgroups (32 rows in two tiles; 3 of one tile are less), four times over
    assert got["decode"] == 256 * 2 * 4 * 4 * (2 * 8 * 256 + 2 * 32 + 4)
    # one user's many rows: one workgroup of four waves with 64 rows of 128 each; several users': that
    # is 4 x 8,324 floats a CU, and 64 rows of 64 two a CU, four times over, 8 x 4,228
    assert got["one"] == 256 * 4 * 4 * (4 * 8 * 256 + 4 * 32 + 4)
    assert got["tree"] == 256 * 2 * 4 * 4 * (4 * 4 * 256 + 4 * 32 + 4)
