"""What can be told of the single-token kernels from their source."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "zkie_b200", "csrc")
FILES = ("q4.cuh", "decode.cu", "decode_moe.cu")


def _code(name):
    """The file without its comments."""
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)


def _body(code, start):
    """From `start` on, the text up to the brace that closes the first one."""
    depth, i = 0, code.index("{", start)
    for j in range(i, len(code)):
        depth += {"{": 1, "}": -1}.get(code[j], 0)
        if depth == 0:
            return code[start:j + 1]
    raise AssertionError("no end")


def test_no_read_only_loads():
    """A kernel that starts while the one before it runs reads what that one
    wrote: not through __ldg, whose data has to stay the same while the kernel
    runs, nor with intrinsics that the compiler may move to before the wait."""
    for name in FILES:
        assert not re.findall(r"__ldg|__ldc[gasv]|__ldlu|ld\.global\.nc|ld\.global", _code(name)), name


def test_kernels_that_start_early_wait_and_restrict_nothing():
    """Every kernel that is launched to overlap the one before it waits for it,
    and none promises that its pointers are read-only (__restrict__)."""
    early = 0
    for name in FILES:
        code = _code(name)
        for m in re.finditer(r"__global__", code):
            text = _body(code, m.start())
            if "let_next_start()" in text or "__grid_constant__" in text:
                early += 1
                assert text.count("wait_for_previous();") == 1 and "__restrict__" not in text, text[:200]
        for m in re.finditer(r"__device__ __forceinline__ [^;{]*\{", code):
            assert "__restrict__" not in m.group(), m.group()
    assert early == 5


def test_nothing_is_asked_for_after_a_wait_that_gave_up():
    """A barrier whose copy never came has no arrival left in its phase: another
    expect_tx would take its count below zero, and another copy would go to a
    slot whose first one is still under way.  Every ring's ask, and every
    later wait, ends at once."""
    wait = _body(_code("q4.cuh"), _code("q4.cuh").index("void barrier_wait"))
    assert wait.index("if (patience.failed) return;") < wait.index("mbarrier.try_wait")
    asks = [(name, m.start()) for name in FILES for m in re.finditer(r"auto ask = ", _code(name))]
    assert len(asks) == 4
    for name, at in asks:
        text = _body(_code(name), at)
        assert re.match(r"auto ask = \[&\]\(\) \{\s*if \(patience\.failed\) return;", text), text[:120]
    # and there is no other place that asks for a copy
    for name in FILES[1:]:
        code = _code(name)
        inside = sum(_body(code, at).count("barrier_expect(") for n, at in asks if n == name)
        assert code.count("barrier_expect(") == inside and code.count("bulk_copy(") == sum(
            _body(code, at).count("bulk_copy(") for n, at in asks if n == name)


# ---- the binding ----------------------------------------------------------------------------------
def test_the_binding_is_built_again_for_another_torch(zk, monkeypatch, tmp_path):
    from zkie_b200 import build
    ran = []

    class Done:
        returncode, stderr = 0, ""

    def run(cmd, **kw):
        ran.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return Done()

    monkeypatch.setattr(build, "CALLS", str(tmp_path / "_calls.so"))
    monkeypatch.setattr(build, "BUILD", str(tmp_path / "_build"))
    if hasattr(build, "CALLS_FOR"):
        monkeypatch.setattr(build, "CALLS_FOR", str(tmp_path / "_build" / "for"))
    monkeypatch.setattr(build.subprocess, "run", run)
    build.build_calls()
    assert len(ran) == 1
    build.build_calls()
    assert len(ran) == 1
    import importlib.metadata
    real = importlib.metadata.version
    monkeypatch.setattr(importlib.metadata, "version", lambda name: "9.9" if name == "torch" else real(name))
    build.build_calls()
    assert len(ran) == 2
    build.build_calls()
    assert len(ran) == 2


def test_the_package_imports_without_its_binding(zk):
    """A binding that does not load stops the per-token calls, not the proofs."""
    import subprocess
    import sys
    code = """
import sys
sys.modules["zkie_b200._calls"] = None
import zkie_b200 as zk
import zkie_b200.deepseek
assert zk.lib.zkie2_q4_words(1, 64, 16, 64, 0) == 136
try:
    zk.decode.choose_token(0, err=0)
except ImportError as e:
    assert "zkie_b200.build" in str(e)
    print("refused")
"""
    res = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=os.path.dirname(os.path.dirname(CSRC)))
    assert res.stdout.strip() == "refused", res.stderr
