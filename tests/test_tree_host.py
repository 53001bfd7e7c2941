"""The tree and cache calls without a GPU: struct layouts, the checks made before
the device is touched, and the Python mirror's refusals."""
import ctypes as C
import os
import shutil
import subprocess
import sys

import pytest

from xwen_amd import _lib

E, CAP, OK = _lib.XS_ERR_ARG, _lib.XS_ERR_CAPACITY, _lib.XS_OK
DEV = 0x7f0000001000
DIMS = _lib.CacheDims(8, 64, 32, 8, 256, 4096)


class Limits(C.Structure):
    _fields_ = [("max_rows", C.c_int64), ("vocab", C.c_int64), ("max_chunks", C.c_int32)]


@pytest.fixture(scope="module")
def host():
    L = C.CDLL(os.environ.get("XS_HOST_LIB") or _lib.LIB_PATH)
    for f in ("dims", "attend", "commit", "evict", "verify_tree"):
        getattr(L, "xs_host_check_" + f).restype = C.c_int
        getattr(L, "xs_host_check_" + f).argtypes = [C.c_void_p] * (1 if f == "dims" else 2)
    return L


def test_structs_match_the_header(tmp_path):
    names = {"xs_verify_tree_args": _lib.VerifyTreeArgs, "xs_cache_dims": _lib.CacheDims, "xs_kv": _lib.Kv,
             "xs_tree_attend_args": _lib.TreeAttendArgs, "xs_cache_commit_args": _lib.CacheCommitArgs,
             "xs_cache_evict_args": _lib.CacheEvictArgs}
    lines = []
    for n, s in names.items():
        lines.append(f'printf("{n} %zu\\n", sizeof({n}));')
        lines += [f'printf("{n}.{f} %zu\\n", offsetof({n}, {f}));' for f, _ in s._fields_]
    src = tmp_path / "t.c"
    src.write_text("#include <stddef.h>\n#include <stdio.h>\n#include \"xsamp.h\"\nint main(void) {" + "\n".join(lines) + "return 0; }")
    exe = tmp_path / "t"
    subprocess.run(["gcc", "-I", os.path.join(_lib.ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = dict(x.rsplit(" ", 1) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for n, s in names.items():
        assert C.sizeof(s) == int(got[n]), n
        for f, _ in s._fields_:
            assert getattr(s, f).offset == int(got[f"{n}.{f}"]), (n, f)


def kv(slot_stride=512, **kw):
    x = _lib.Kv(DEV, DEV, 4096 * 512, slot_stride, 64)
    for k, v in kw.items():
        setattr(x, k, v)
    return x


def attend(**kw):
    a = _lib.TreeAttendArgs(dtype=_lib.BF16, head_dim=64, seqs=4, nodes=16, q_heads=16, kv_heads=8, q=DEV, q_seq_stride=16 * 1024,
                            q_node_stride=1024, q_head_stride=64, cache=kv(), capacity=4096, len=DEV, fresh=kv(), parent=DEV,
                            scale=0.1, out=DEV + 4096, out_seq_stride=16 * 1024, out_node_stride=1024, out_head_stride=64,
                            seq_status=DEV)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_sizes_of_a_context(host):
    def chk(**kw):
        d = _lib.CacheDims(8, 64, 32, 8, 256, 4096)
        for k, v in kw.items():
            setattr(d, k, v)
        return host.xs_host_check_dims(C.byref(d))
    assert chk() == OK and host.xs_host_check_dims(None) == E
    assert chk(max_seqs=0) == E and chk(max_nodes=0) == E and chk(max_nodes=65) == E and chk(q_heads=0) == E
    assert chk(kv_heads=0) == E and chk(head_dim=7) == E and chk(head_dim=264) == E and chk(capacity=0) == E
    assert chk(max_seqs=1 << 20) == CAP and chk(kv_heads=33) == CAP and chk(capacity=1 << 40) == CAP and chk(q_heads=1 << 20) == CAP


def test_attend_checks(host):
    chk = lambda **kw: host.xs_host_check_attend(C.byref(DIMS), C.byref(attend(**kw)))
    assert chk() == OK
    assert host.xs_host_check_attend(None, C.byref(attend())) == E and host.xs_host_check_attend(C.byref(DIMS), None) == E
    for f in ("q", "len", "parent", "out", "seq_status"):
        assert chk(**{f: None}) == E, f
    assert chk(n_nodes=DEV, lse=DEV, max_len=4096) == OK
    assert chk(dtype=2) == E and chk(dtype=-1) == E
    assert chk(head_dim=0) == E and chk(head_dim=60) == E and chk(head_dim=264) == E
    assert chk(seqs=-1) == E and chk(seqs=0) == OK and chk(seqs=9) == CAP
    assert chk(nodes=0) == E and chk(nodes=65) == E
    assert chk(q_heads=12) == E and chk(q_heads=0) == E and chk(kv_heads=0) == E and chk(q_heads=48) == CAP
    assert chk(kv_heads=16) == CAP and chk(capacity=0) == E and chk(capacity=4097) == CAP
    assert chk(max_len=-1) == E and chk(max_len=4097) == E
    assert chk(q=DEV + 8) == E and chk(out=DEV + 2) == E and chk(out=DEV) == E
    assert chk(q_node_stride=1020) == E and chk(q_head_stride=-64) == E and chk(q_seq_stride=0) == OK
    assert chk(out_head_stride=0) == E and chk(out_node_stride=512) == E and chk(out_seq_stride=1024) == E
    assert chk(cache=kv(k=None)) == E and chk(cache=kv(v=DEV + 4)) == E and chk(cache=kv(12)) == E and chk(fresh=kv(-8)) == E
    assert chk(cache=kv(seq_stride=1 << 62)) == E and chk(fresh=kv(head_stride=1 << 61)) == E
    assert chk(fresh=kv(0)) == OK
    small = _lib.CacheDims(8, 4, 32, 8, 32, 4096)
    assert host.xs_host_check_attend(C.byref(small), C.byref(attend(nodes=4))) == CAP
    small = _lib.CacheDims(8, 4, 32, 8, 64, 4096)
    assert host.xs_host_check_attend(C.byref(small), C.byref(attend())) == CAP


def commit(**kw):
    a = _lib.CacheCommitArgs(dtype=_lib.F16, head_dim=64, seqs=4, nodes=16, q_heads=16, kv_heads=8, cache=kv(), capacity=4096, len=DEV,
                             fresh=kv(), path=DEV, path_ld=16, n_path=DEV, new_len=DEV + 64, slot_ld=4096, seq_status=DEV)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_commit_checks(host):
    chk = lambda **kw: host.xs_host_check_commit(C.byref(DIMS), C.byref(commit(**kw)))
    w = dict(q=DEV, q_seq_stride=16 * 1024, q_node_stride=1024, q_head_stride=64, lse=DEV, mass=DEV, new_mass=DEV, scale=1.0)
    p = dict(next_pos=DEV, pos=DEV, new_next_pos=DEV + 64)
    assert chk() == OK and chk(**w) == OK and chk(**p) == OK and chk(**w, **p) == OK
    assert host.xs_host_check_commit(None, C.byref(commit())) == E and host.xs_host_check_commit(C.byref(DIMS), None) == E
    for f in ("len", "path", "n_path", "new_len", "seq_status"):
        assert chk(**{f: None}) == E, f
    for f in ("q", "lse", "mass", "new_mass"):
        assert chk(**{**w, f: None}) == E, f
    for f in p:
        assert chk(**{**p, f: None}) == E, f
    assert chk(new_len=DEV) == E and chk(**{**p, "new_next_pos": DEV}) == E
    assert chk(new_len=DEV + 12) == E and chk(new_len=DEV + 16) == OK and chk(new_len=DEV - 12) == E  # [4] int32 each
    assert chk(path_ld=15) == E and chk(slot_ld=4095) == E and chk(slot_ld=1 << 60) == E and chk(path_ld=1 << 40) == E
    assert chk(cache=kv(0)) == E and chk(cache=kv(64)) == E and chk(fresh=kv(0)) == OK
    assert chk(**{**w, "q": DEV + 2}) == E and chk(**{**w, "q_head_stride": 4}) == E
    assert chk(nodes=0) == E and chk(q_heads=9) == E and chk(max_len=5000) == E and chk(seqs=9) == CAP


def evict(**kw):
    a = _lib.CacheEvictArgs(dtype=_lib.BF16, head_dim=64, seqs=4, kv_heads=8, cache=kv(), capacity=4096, len=DEV, mass=DEV, new_mass=DEV,
                            pos=DEV, new_pos=DEV, slot_ld=4096, next_pos=DEV, keep=1000, sinks=4, recent=64, new_len=DEV + 64,
                            seq_status=DEV)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_evict_checks(host):
    chk = lambda **kw: host.xs_host_check_evict(C.byref(DIMS), C.byref(evict(**kw)))
    assert chk() == OK
    assert host.xs_host_check_evict(None, C.byref(evict())) == E and host.xs_host_check_evict(C.byref(DIMS), None) == E
    for f in ("len", "mass", "new_mass", "pos", "new_pos", "next_pos", "new_len", "seq_status"):
        assert chk(**{f: None}) == E, f
    assert chk(new_len=DEV) == E and chk(new_mass=DEV + 4096) == E and chk(new_mass=DEV + 4096, new_pos=DEV + 4096) == OK
    assert chk(keep=0) == E and chk(sinks=-1) == E and chk(recent=-1) == E
    assert chk(keep=68) == OK and chk(keep=67) == E and chk(sinks=1 << 62, recent=1 << 62) == E and chk(keep=1 << 62) == OK
    assert chk(slot_ld=4095) == E and chk(slot_ld=1 << 62) == E
    assert chk(cache=kv(0)) == E and chk(cache=kv(head_stride=0)) == E and chk(cache=kv(seq_stride=512)) == E
    assert chk(capacity=5000) == CAP and chk(head_dim=4) == E and chk(dtype=7) == E


def test_verify_tree_checks(host):
    lim = Limits(64, 300_000, 19)

    def chk(**kw):
        a = _lib.VerifyTreeArgs(logits=DEV, seqs=4, nodes=16, ld=248_320, width=248_320, enc=248_320, params=DEV, uniforms=DEV,
                                tokens=DEV, parent=DEV, row_token=DEV, row_status=DEV, accepted=DEV, path=DEV, committed=DEV,
                                n_committed=DEV, seq_status=DEV)
        for k, v in kw.items():
            setattr(a, k, v)
        return host.xs_host_check_verify_tree(C.byref(lim), C.byref(a))
    assert chk() == OK and chk(seqs=0) == OK and chk(n_nodes=DEV, budget=DEV, done_after=DEV) == OK
    for f in ("logits", "params", "uniforms", "tokens", "parent", "row_token", "row_status", "accepted", "path", "committed",
              "n_committed", "seq_status"):
        assert chk(**{f: None}) == E, f
    assert chk(nodes=0) == E and chk(nodes=65, seqs=1) == E and chk(seqs=-1) == E and chk(seqs=5) == CAP
    assert chk(n_eog=1) == E and chk(n_eog=-1) == E and chk(n_eog=1, eog=DEV) == OK and chk(k_max=-1) == E
    assert chk(ld=248_322) == E and chk(logits=DEV + 4) == E
    assert host.xs_host_check_verify_tree(None, None) == E


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
    r = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-p", "no:cacheprovider", "-k", "checks and not asan or sizes",
                        os.path.abspath(__file__)], cwd=_lib.ROOT, env=env, capture_output=True, text=True, timeout=600)
    tail = (r.stdout + r.stderr)[-4000:]
    assert r.returncode == 0 and " passed" in r.stdout, tail
    assert "AddressSanitizer" not in r.stderr and "runtime error:" not in r.stderr, tail


def test_calls_without_a_context():
    lib = _lib.load()
    assert lib.xs_tree_attend(None, C.byref(attend())) == E
    assert lib.xs_cache_commit(None, C.byref(commit())) == E
    assert lib.xs_cache_evict(None, C.byref(evict())) == E
    assert lib.xs_verify_tree(None, C.byref(_lib.VerifyTreeArgs())) == E
    assert lib.xs_cache_set_stream(None, None) == E and lib.xs_cache_destroy(None) == OK
    assert lib.xs_cache_create(0, C.byref(DIMS), None) == E
    h = C.c_void_p(1)
    bad = _lib.CacheDims(8, 65, 32, 8, 256, 4096)
    assert lib.xs_cache_create(0, C.byref(bad), C.byref(h)) == E and not h.value


def test_the_mirror_refuses_what_does_not_fit():
    torch = pytest.importorskip("torch")
    from xwen_amd import tree

    class Ctx:
        device = 0

    t = torch.zeros((2, 3, 4, 64), dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="not on the context's device"):
        tree.tree_attend(Ctx(), t, t, t, i, t, t, i)
    with pytest.raises(ValueError, match="bfloat16 or float16"):
        tree.tree_attend(Ctx(), t.float(), t, t, i, t, t, i)
    with pytest.raises(ValueError):
        tree.cache_commit(Ctx(), t, t, i, t, t, i, i)
    with pytest.raises(ValueError):
        tree.cache_evict(Ctx(), t, t, i, i, i, i, 2)
