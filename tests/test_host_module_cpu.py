"""CPU: what the compiled host part of the bounded-cache calls (_fa_b200_host.so) is needed for, and when it is built."""
import importlib.util
import os
import re
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "flash-attention-das_b200")


@pytest.fixture(scope="module")
def builder():
    spec = importlib.util.spec_from_file_location("_fa_build", os.path.join(PKG, "build.py"))
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    b.build()
    return b


def package(tmp_path, host=False):
    """A copy of the package's Python files beside the built library, without the host module."""
    to = tmp_path / "pkg"
    shutil.copytree(PKG, to, ignore=shutil.ignore_patterns("*.so", "build", "csrc", "__pycache__"))
    os.symlink(os.path.join(PKG, "libfa_b200.so"), to / "libfa_b200.so")
    if host:
        os.symlink(os.path.join(PKG, "_fa_b200_host.so"), to / "_fa_b200_host.so")
    return str(to)


def run(path, code, **env):
    return subprocess.run([sys.executable, "-c", f"import sys; sys.path.insert(0, {path!r})\n" + code], capture_output=True, text=True,
                          env={**os.environ, **env})


PLAIN = """
import torch
import flash_attn as fa, flash_attn_2_cuda as c
assert c.__file__.startswith(sys.path[0])
assert c.lib().fa_b200_abi_version() == 2
c.set_profile_events(None, None)
try:
    fa.flash_attn_func(*[torch.zeros(1, 8, 2, 128, dtype=torch.bfloat16)] * 3)
except (RuntimeError, ValueError, NotImplementedError) as e:   # CPU tensors: refused as such, by the call itself
    assert not isinstance(e, ImportError)
"""
BOUNDED = """
try:
    fa.kvcache_page_bounds(torch.zeros(4, 64, 2, 128, dtype=torch.bfloat16), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))
except ImportError as e:
    print("REFUSED", e)
"""


def test_other_entry_points_do_not_need_it(builder, tmp_path):
    r = run(package(tmp_path), PLAIN + BOUNDED)
    assert r.returncode == 0, r.stderr
    assert "REFUSED" in r.stdout and "not found" in r.stdout


def test_a_library_without_the_bounded_calls(builder, tmp_path):
    """FA_B200_LIB naming a library with every other function."""
    names = set(re.findall(r"_lib\.(fa_b200_\w+)", open(os.path.join(PKG, "flash_attn_2_cuda.py")).read()))
    names -= {n for n in names if re.search("page_bounds|page_select|decode_budget|token_weights|kv_evict", n)}
    src, so = tmp_path / "old.c", tmp_path / "old.so"
    src.write_text("".join("long %s(void) { return 2; }\n" % n for n in sorted(names)))
    subprocess.run(["gcc", "-shared", "-fPIC", str(src), "-o", str(so)], check=True)
    r = run(package(tmp_path, host=True), PLAIN + BOUNDED, FA_B200_LIB=str(so))
    assert r.returncode == 0, r.stderr
    assert "REFUSED" in r.stdout and "fa_b200_page_bounds" in r.stdout


def test_it_is_loaded_once_by_the_first_bounded_call(builder, tmp_path):
    r = run(package(tmp_path, host=True), PLAIN + """
assert "_host" not in vars(c)
import threading
got = []
ts = [threading.Thread(target=lambda: got.append(c.page_select)) for _ in range(8)]
[t.start() for t in ts]; [t.join() for t in ts]
assert len(set(map(id, got))) == 1 and c._host.page_select is got[0] and vars(c)["kv_evict"] is c._host.kv_evict
assert not hasattr(c, "no_such_call")
""")
    assert r.returncode == 0, r.stderr


def test_it_is_built_for_one_torch_in_full(builder, tmp_path):
    """A pre-release differs from the release of its number, and from another pre-release; the module's own torch never does."""
    import torch
    import flash_attn_2_cuda
    assert torch.__version__ in flash_attn_2_cuda._host.BUILT_FOR and flash_attn_2_cuda._host.BUILT_FOR == builder.host_key()
    path = package(tmp_path, host=True)
    release = torch.__version__.split("+")[0]
    for other in (release + "a0+git1234567", release + ".dev20260101", release if "+" in torch.__version__ else release + "+vendor"):
        r = run(path, f"import torch; torch.__version__ = {other!r}\n" + PLAIN + BOUNDED)
        assert r.returncode == 0, r.stderr
        assert "REFUSED" in r.stdout and other in r.stdout


def test_a_module_of_another_torch_is_rebuilt(builder, tmp_path, monkeypatch):
    assert not builder.needs_build(builder.OUT_HOST)
    monkeypatch.setattr(builder, "HOST_KEY", str(tmp_path / "key"))
    assert builder.needs_build(builder.OUT_HOST)                    # nobody knows what it was built for
    (tmp_path / "key").write_text(builder.host_key())
    assert not builder.needs_build(builder.OUT_HOST)
    monkeypatch.setattr("torch.__version__", "2.99.0a0+git1234567")
    assert "2.99.0a0+git1234567" in builder.host_key() and builder.needs_build(builder.OUT_HOST)
    assert not builder.needs_build(builder.OUT)


def test_the_library_is_built_without_torch(builder, monkeypatch, capsys):
    """The C ABI has callers without Python packages."""
    made = []
    monkeypatch.setattr(builder, "build_host", lambda force=False: made.append(force))
    monkeypatch.setattr("importlib.util.find_spec", lambda name: None)
    assert builder.build() == builder.OUT and made == [] and "no torch" in capsys.readouterr().err
    monkeypatch.undo()
    monkeypatch.setattr(builder, "build_host", lambda force=False: made.append(force))
    assert builder.build() == builder.OUT and made == [False]
