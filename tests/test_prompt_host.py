"""The prompt's and the 8-bit cache's calls without a GPU: struct layouts, the checks made
before the device is touched, the Python mirror's refusals, and what the calls leave of the
thread's current device."""
import ctypes as C
import os
import shutil
import subprocess
import sys

import pytest

from tests.test_tree_device import child, runtime  # noqa: F401 (a fixture)
from tests.test_tree_host import kv
from xwen_amd import _lib

E, CAP, OK = _lib.XS_ERR_ARG, _lib.XS_ERR_CAPACITY, _lib.XS_OK
DEV = 0x7f0000001000
DIMS = _lib.CacheDims(8, 64, 32, 8, 256, 4096)


@pytest.fixture(scope="module")
def host():
    L = C.CDLL(os.environ.get("XS_HOST_LIB") or _lib.LIB_PATH)
    for f, n in (("rotate", 1), ("prompt", 1), ("append8", 2), ("attend8", 2)):
        getattr(L, "xs_host_check_" + f).restype = C.c_int
        getattr(L, "xs_host_check_" + f).argtypes = [C.c_void_p] * n
    return L


def test_structs_match_the_header(tmp_path):
    names = {"xs_qk_rotate_args": _lib.QkRotateArgs, "xs_prompt_attend_args": _lib.PromptAttendArgs, "xs_kv8": _lib.Kv8,
             "xs_cache_append8_args": _lib.CacheAppend8Args, "xs_tree_attend8_args": _lib.TreeAttend8Args}
    lines = []
    for n, s in names.items():
        lines.append(f'printf("{n} %zu\\n", sizeof({n}));')
        lines += [f'printf("{n}.{f} %zu\\n", offsetof({n}, {f}));' for f, _ in s._fields_]
    lines += ['printf("block %d\\n", XS_CACHE8_BLOCK);', 'printf("rot %d\\n", 10 * XS_ROT_HALVES + XS_ROT_NEIGHBOURS);']
    src = tmp_path / "t.c"
    src.write_text("#include <stddef.h>\n#include <stdio.h>\n#include \"xsamp.h\"\nint main(void) {" + "\n".join(lines) + "return 0; }")
    exe = tmp_path / "t"
    subprocess.run(["gcc", "-I", os.path.join(_lib.ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = dict(x.rsplit(" ", 1) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for n, s in names.items():
        assert C.sizeof(s) == int(got[n]), n
        for f, _ in s._fields_:
            assert getattr(s, f).offset == int(got[f"{n}.{f}"]), (n, f)
    assert int(got["block"]) == _lib.CACHE8_BLOCK and int(got["rot"]) == 10 * _lib.ROT_HALVES + _lib.ROT_NEIGHBOURS


def rotate(**kw):
    a = _lib.QkRotateArgs(dtype=_lib.BF16, head_dim=64, tokens=100, q_heads=16, kv_heads=4, q=DEV, q_token_stride=1024, q_head_stride=64,
                          k=DEV + (1 << 20), k_token_stride=256, k_head_stride=64, eps=1e-6, rot_dim=64, inv_freq=DEV, pos=DEV,
                          q_out=DEV + (2 << 20), q_out_token_stride=1024, q_out_head_stride=64, k_out=DEV + (3 << 20),
                          k_out_token_stride=256, k_out_head_stride=64)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_rotate_checks(host):
    chk = lambda **kw: host.xs_host_check_rotate(C.byref(rotate(**kw)))
    assert chk() == OK and host.xs_host_check_rotate(None) == E
    assert chk(dtype=2) == E and chk(head_dim=60) == E and chk(head_dim=264) == E and chk(head_dim=0) == E
    assert chk(tokens=-1) == E and chk(tokens=0, q=None) == OK and chk(q_heads=-1) == E and chk(kv_heads=1 << 20) == CAP
    for f in ("q", "k", "q_out", "k_out", "pos", "inv_freq"):
        assert chk(**{f: None}) == E, f
    assert chk(rot_dim=0, pos=None, inv_freq=None) == OK
    assert chk(rot_dim=-16) == E and chk(rot_dim=80) == E and chk(rot_dim=8) == E and chk(rot_dim=24) == E and chk(rot_dim=48) == OK
    assert chk(rot_dim=24, pairs=_lib.ROT_NEIGHBOURS) == OK and chk(rot_dim=12, pairs=_lib.ROT_NEIGHBOURS) == E and chk(pairs=2) == E
    assert chk(eps=-1.0) == E and chk(eps=float("nan")) == E and chk(eps=0.0) == OK
    assert chk(q_weight=DEV) == E and chk(k_weight=DEV) == E and chk(q_weight=DEV, k_weight=DEV) == OK
    assert chk(q_weight=DEV + 4, k_weight=DEV) == E
    assert chk(q_heads=0, q=None, q_out=None, k_weight=DEV) == OK and chk(kv_heads=0, k=None, k_out=None, q_weight=DEV) == OK
    assert chk(q_heads=0, kv_heads=0, q=None, k=None) == OK
    assert chk(q=DEV + 8) == E and chk(k_out=DEV + 2) == E and chk(q_token_stride=1020) == E and chk(k_head_stride=-64) == E
    assert chk(q_token_stride=0) == OK and chk(q_out_token_stride=0) == E and chk(q_out_head_stride=32) == E
    assert chk(q_token_stride=1 << 60) == E
    # in place with the same strides only; no other overlap that shows in the pointers
    assert chk(q_out=DEV) == OK and chk(q_out=DEV, q_out_token_stride=2048) == E
    assert chk(q_out=DEV + (1 << 20)) == E and chk(k_out=DEV) == E and chk(k_out=DEV + (2 << 20)) == E


def prompt(**kw):
    a = _lib.PromptAttendArgs(dtype=_lib.F16, head_dim=64, seqs=3, tokens=100, q_heads=16, kv_heads=4, q=DEV, q_token_stride=1024,
                              q_head_stride=64, k=DEV + (1 << 20), v=DEV + (2 << 20), kv_token_stride=256, kv_head_stride=64, start=DEV,
                              scale=0.1, out=DEV + (3 << 20), out_token_stride=1024, out_head_stride=64, seq_status=DEV)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_prompt_checks(host):
    chk = lambda **kw: host.xs_host_check_prompt(C.byref(prompt(**kw)))
    assert chk() == OK and host.xs_host_check_prompt(None) == E
    for f in ("q", "k", "v", "start", "out", "seq_status"):
        assert chk(**{f: None}) == E, f
    assert chk(seqs=0, start=None) == OK and chk(tokens=0, q=None, k=None, v=None, out=None) == OK and chk(tokens=0, start=None) == E
    assert chk(dtype=2) == E and chk(head_dim=60) == E and chk(head_dim=0) == E and chk(head_dim=264) == E and chk(head_dim=72) == E
    assert chk(head_dim=56) == OK
    assert chk(seqs=-1) == E and chk(tokens=-1) == E and chk(q_heads=18) == E and chk(q_heads=0) == E and chk(kv_heads=0) == E
    assert chk(seqs=70000) == CAP and chk(tokens=(1 << 28) + 1) == CAP and chk(q_heads=8192) == CAP and chk(kv_token_stride=(1 << 24) + 8) == CAP
    assert chk(q=DEV + 8) == E and chk(k=DEV + 4) == E and chk(v=DEV + 2) == E and chk(out=DEV + 8) == E
    assert chk(out=DEV) == E and chk(out=DEV + (1 << 20)) == E and chk(out=DEV + (2 << 20)) == E
    assert chk(q_token_stride=1020) == E and chk(kv_head_stride=-64) == E and chk(out_token_stride=512) == E and chk(out_head_stride=0) == E
    assert chk(kv_token_stride=0, kv_head_stride=0, q_token_stride=0) == OK and chk(q_head_stride=1 << 60) == E


def kv8(**kw):
    a = _lib.Kv8(DEV, DEV + (1 << 24), 4096 * 512, 512, 64, DEV, DEV + 4096, 128)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def append(**kw):
    a = _lib.CacheAppend8Args(dtype=_lib.BF16, head_dim=64, seqs=4, rows=16, kv_heads=8, cache=kv8(), capacity=4096, len=DEV, fresh=kv(),
                              new_len=DEV + 64, seq_status=DEV)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_append_checks(host):
    chk = lambda **kw: host.xs_host_check_append8(C.byref(DIMS), C.byref(append(**kw)))
    assert chk() == OK and host.xs_host_check_append8(None, C.byref(append())) == E and host.xs_host_check_append8(C.byref(DIMS), None) == E
    for f in ("len", "new_len", "seq_status"):
        assert chk(**{f: None}) == E, f
    assert chk(path=DEV, path_ld=16, n_path=DEV) == OK and chk(path=DEV, path_ld=15) == E and chk(n_path=DEV) == OK
    assert chk(start=DEV, tokens=100) == OK and chk(start=DEV, tokens=100, n_path=DEV) == E and chk(start=DEV, path=DEV, path_ld=16) == E
    assert chk(start=DEV, tokens=100, fresh=kv(seq_stride=-8)) == OK and chk(fresh=kv(seq_stride=-8)) == E
    assert chk(start=DEV, tokens=0, fresh=kv(k=None)) == OK and chk(rows=0, fresh=kv(k=None)) == OK and chk(fresh=kv(k=None)) == E
    assert chk(dtype=2) == E and chk(head_dim=72) == E and chk(head_dim=8) == E and chk(head_dim=0) == E and chk(head_dim=272) == E
    assert chk(seqs=0, len=None) == OK and chk(seqs=9) == CAP and chk(rows=-1) == E and chk(rows=1 << 40) == CAP and chk(tokens=-1) == E
    assert chk(kv_heads=9) == CAP and chk(capacity=4097) == CAP and chk(capacity=0) == E
    assert chk(new_len=DEV) == E and chk(new_len=DEV + 8) == E
    assert chk(cache=kv8(k=None)) == E and chk(cache=kv8(v_exp=None)) == E and chk(cache=kv8(k=DEV + 8)) == E
    assert chk(cache=kv8(slot_stride=520)) == E and chk(cache=kv8(slot_stride=0)) == E and chk(cache=kv8(exp_ld=127)) == E
    assert chk(cache=kv8(exp_ld=1 << 61)) == E and chk(cache=kv8(head_stride=48)) == E


def attend8(**kw):
    a = _lib.TreeAttend8Args(dtype=_lib.BF16, head_dim=64, seqs=4, nodes=16, q_heads=16, kv_heads=8, q=DEV, q_seq_stride=16 * 1024,
                             q_node_stride=1024, q_head_stride=64, cache=kv8(), capacity=4096, len=DEV, fresh=kv(), parent=DEV,
                             scale=0.1, out=DEV + 4096, out_seq_stride=16 * 1024, out_node_stride=1024, out_head_stride=64, seq_status=DEV)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_attend8_checks(host):
    chk = lambda **kw: host.xs_host_check_attend8(C.byref(DIMS), C.byref(attend8(**kw)))
    assert chk() == OK and host.xs_host_check_attend8(None, C.byref(attend8())) == E and host.xs_host_check_attend8(C.byref(DIMS), None) == E
    for f in ("q", "len", "parent", "out", "seq_status"):
        assert chk(**{f: None}) == E, f
    assert chk(n_nodes=DEV, lse=DEV, max_len=4096) == OK and chk(max_len=4097) == E and chk(max_len=-1) == E
    assert chk(dtype=2) == E and chk(head_dim=72) == E and chk(head_dim=264) == E and chk(nodes=0) == E and chk(nodes=65) == E
    assert chk(seqs=0, q=None) == OK and chk(seqs=9) == CAP and chk(q_heads=12) == E and chk(q_heads=48) == CAP and chk(kv_heads=16) == CAP
    assert chk(q=DEV + 8) == E and chk(out=DEV) == E and chk(q_node_stride=1020) == E and chk(out_head_stride=0) == E
    assert chk(cache=kv8(v=None)) == E and chk(cache=kv8(k_exp=None)) == E and chk(cache=kv8(slot_stride=8)) == E and chk(cache=kv8(exp_ld=1)) == E
    assert chk(cache=kv8(slot_stride=(1 << 25) + 16)) == CAP and chk(cache=kv8(slot_stride=1 << 25)) == OK
    assert chk(cache=kv8(slot_stride=0)) == OK and chk(fresh=kv(v=DEV + 4)) == E and chk(fresh=kv(0)) == OK


def test_the_checks_under_asan_and_ubsan():
    """The checks above against the sanitized host build, in a child process."""
    if os.environ.get("XS_HOST_LIB"):
        pytest.skip("this is the child")
    rt = subprocess.run(["gcc", "-print-file-name=libasan.so"], capture_output=True, text=True).stdout.strip() if shutil.which("gcc") else ""
    if not os.path.isabs(rt) or not os.path.exists(rt) or not shutil.which("make"):
        pytest.skip("gcc's AddressSanitizer runtime is not installed")
    oracle = os.path.join(_lib.ROOT, "oracle")
    subprocess.run(["make", "-s", "-C", oracle, "asan"], check=True)
    env = dict(os.environ, LD_PRELOAD=rt, ASAN_OPTIONS="detect_leaks=0:halt_on_error=1:abort_on_error=1",
               UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1",
               XS_ORACLE_LIB=os.path.join(oracle, "_build", "asan", "libxs_oracle.so"),
               XS_HOST_LIB=os.path.join(oracle, "_build", "asan", "libxs_host.so"))
    r = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-p", "no:cacheprovider", "-k", "checks and not asan",
                        os.path.abspath(__file__)], cwd=_lib.ROOT, env=env, capture_output=True, text=True, timeout=600)
    tail = (r.stdout + r.stderr)[-4000:]
    assert r.returncode == 0 and " passed" in r.stdout, tail
    assert "AddressSanitizer" not in r.stderr and "runtime error:" not in r.stderr, tail


def test_the_mirror_refuses_what_does_not_fit():
    torch = pytest.importorskip("torch")
    from xwen_amd import cache8, prompt as px

    class Ctx:
        device = 0

    t = torch.zeros((3, 4, 64), dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="not on the context's device"):
        px.qk_rotate(Ctx(), t, t)
    with pytest.raises(ValueError, match="bfloat16 or float16"):
        px.qk_rotate(Ctx(), t.float(), t.float())
    with pytest.raises(ValueError, match="both None"):
        px.qk_rotate(Ctx(), None, None)
    with pytest.raises(ValueError, match="go together"):
        px.qk_rotate(Ctx(), t, t, i)
    with pytest.raises(ValueError, match="not on the context's device"):
        px.prompt_attend(Ctx(), t, t, t, i)
    c8, e8 = torch.zeros((2, 64, 4, 64), dtype=torch.float8_e4m3fn), torch.zeros((2, 4, 2), dtype=torch.uint8)
    f = torch.zeros((2, 3, 4, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="not on the context's device"):
        cache8.cache_append8(Ctx(), c8, c8, e8, e8, i, f, f)
    with pytest.raises(ValueError, match="not on the context's device"):
        cache8.tree_attend8(Ctx(), f, c8, c8, e8, e8, i, f, f, i)


def test_calls_without_a_context():
    lib = _lib.load()
    assert lib.xs_qk_rotate(None, C.byref(rotate())) == E and lib.xs_prompt_attend(None, C.byref(prompt())) == E
    assert lib.xs_cache_append8(None, C.byref(append())) == E and lib.xs_tree_attend8(None, C.byref(attend8())) == E


CALLS = """
def more(h):
    r = _lib.QkRotateArgs(dtype=_lib.BF16, head_dim=64, tokens=100, q_heads=16, kv_heads=8, q=P, q_token_stride=1024, q_head_stride=64,
                          k=P + (1 << 20), k_token_stride=512, k_head_stride=64, rot_dim=64, inv_freq=P, pos=P, q_out=P,
                          q_out_token_stride=1024, q_out_head_stride=64, k_out=P + (1 << 20), k_out_token_stride=512, k_out_head_stride=64)
    p = _lib.PromptAttendArgs(dtype=_lib.F16, head_dim=64, seqs=3, tokens=100, q_heads=16, kv_heads=8, q=P, q_token_stride=1024,
                              q_head_stride=64, k=P + (1 << 20), v=P + (2 << 20), kv_token_stride=512, kv_head_stride=64, start=P,
                              scale=0.1, out=P + (3 << 20), out_token_stride=1024, out_head_stride=64, seq_status=P)
    c8 = _lib.Kv8(P, P + (1 << 24), 64 * 512, 512, 64, P, P + 4096, 2)
    a = _lib.CacheAppend8Args(dtype=_lib.BF16, head_dim=64, seqs=4, rows=16, kv_heads=8, cache=c8, capacity=64, len=P, fresh=kv(),
                              new_len=P + 64, seq_status=P)
    t = _lib.TreeAttend8Args(dtype=_lib.BF16, head_dim=64, seqs=4, nodes=16, q_heads=16, kv_heads=8, q=P, q_seq_stride=16 * 1024,
                             q_node_stride=1024, q_head_stride=64, cache=c8, capacity=64, len=P, fresh=kv(), parent=P, scale=0.1,
                             out=P + 4096, out_seq_stride=16 * 1024, out_node_stride=1024, out_head_stride=64, seq_status=P)
    return [(lib.xs_qk_rotate, r), (lib.xs_prompt_attend, p), (lib.xs_cache_append8, a), (lib.xs_tree_attend8, t)]
"""


def test_calls_leave_the_current_device(runtime):  # noqa: F811
    child(runtime, CALLS + """
rc, h = cache()
assert rc == 0
for now in (0, 1):
    rt.hipSetDevice(now)
    for call, args in more(h):
        before = rt.fake_launches()
        assert call(h, C.byref(args)) == 0 and rt.fake_launches() > before, call
        assert device() == now, (call.__name__, now, device())
print("done")
""")


def test_launches_past_32_bits_are_refused(runtime):  # noqa: F811
    """2^32 work-items and more of one launch; what is just below them is launched."""
    child(runtime, CALLS + """
rc, h = cache((65536, 64, 4096, 64, 256, 1 << 20))
assert rc == 0
(rot, r), (pr, p), (ap, a), (at, t) = more(h)
r.tokens, r.q_heads, r.q_token_stride, r.q_out_token_stride = 1 << 22, 1024, 65536, 65536
r.k_token_stride = r.k_out_token_stride = 512
for tokens, want in ((1 << 24, _lib.XS_ERR_CAPACITY), (1 << 20, 0)):
    r.tokens = tokens
    assert rot(h, C.byref(r)) == want, tokens
    assert rt.fake_work_items() < 1 << 32
p.q_heads, p.kv_heads, p.q_token_stride, p.out_token_stride = 4096, 4096, 1 << 18, 1 << 18
p.kv_token_stride = 1 << 18
for tokens, want in ((1 << 30, _lib.XS_ERR_CAPACITY), (1 << 16, 0)):
    p.tokens = tokens
    assert pr(h, C.byref(p)) == want, tokens
    assert rt.fake_work_items() < 1 << 32
a.seqs, a.kv_heads, a.capacity, a.rows = 65536, 64, 1 << 20, 1 << 20
a.len, a.new_len = P, P + (1 << 20)
a.cache.seq_stride, a.cache.slot_stride, a.cache.head_stride, a.cache.exp_ld = 1 << 32, 1 << 12, 64, 1 << 15
assert ap(h, C.byref(a)) == _lib.XS_ERR_CAPACITY
a.rows = 1
assert ap(h, C.byref(a)) == 0 and rt.fake_work_items() < 1 << 32
print("done")
""")


def test_calls_of_any_size_within_a_context(runtime):  # noqa: F811
    """Every attend8 call within a context's sizes has room for its partial results."""
    child(runtime, """
import random
rng = random.Random(2)
for _ in range(1200):
    kv = rng.choice([1, 2, 3, 8, 16])
    dims = dict(seqs=rng.choice([1, 2, 7, 64, 900]), nodes=rng.choice([1, 2, 5, 16, 33, 64]), g=rng.choice([1, 2, 4, 7, 16]),
                dim=rng.choice([16, 64, 80, 128, 144, 256]), cap=rng.choice([1, 64, 300, 480, 512, 700, 2000, 9000, 70000, 1 << 20]))
    rc, h = cache((dims["seqs"], dims["nodes"], kv * dims["g"], kv, dims["dim"], dims["cap"]))
    assert rc == 0
    for _ in range(12):
        k = rng.randint(1, kv)
        q = k * rng.randint(1, kv * dims["g"] // k)
        seqs, nodes, cap = rng.randint(1, dims["seqs"]), rng.randint(1, dims["nodes"]), rng.randint(1, dims["cap"])
        dim = 16 * rng.randint(1, dims["dim"] // 16)
        if rng.random() < 0.5:
            k, q, seqs, nodes, cap, dim = kv, kv * dims["g"], dims["seqs"], dims["nodes"], dims["cap"], dims["dim"]
        c8 = _lib.Kv8(P, P, cap * k * 256, k * 256, 256, P, P, (cap + 31) // 32)
        a = _lib.TreeAttend8Args(dtype=rng.randint(0, 1), head_dim=dim, seqs=seqs, nodes=nodes, q_heads=q, kv_heads=k, q=P,
                                 q_seq_stride=nodes * q * 256, q_node_stride=q * 256, q_head_stride=256, cache=c8, capacity=cap, len=P,
                                 fresh=_lib.Kv(P, P, nodes * k * 256, k * 256, 256), parent=P, scale=0.1, out=P + 4096,
                                 out_seq_stride=nodes * q * 256, out_node_stride=q * 256, out_head_stride=256, seq_status=P)
        assert lib.xs_tree_attend8(h, C.byref(a)) == 0, (dims, kv, seqs, nodes, q, k, dim, cap)
    lib.xs_cache_destroy(h)
print("done")
""")
