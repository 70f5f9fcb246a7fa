"""What `make` would run, on the CPU: nothing is compiled here."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "uemda_amd", "csrc")


def commands(*args):
    res = subprocess.run(["make", "-n", "-C", CSRC, *args], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    return res.stdout


def test_the_c_library_alone_needs_neither_torch_nor_python():
    out = commands("-B", "PY=/nonexistent/python3")
    assert "libuemda_hip.so" in out and "grouped.hip" in out and "_host.so" not in out
    assert "_host.so" in commands("-B", "host") and "-ltorch_python" in commands("-B", "host")


def test_build_makes_both(monkeypatch):
    from uemda_amd import _lib
    seen = []
    monkeypatch.setattr(_lib.subprocess, "run", lambda cmd, **kw: seen.append(cmd) or type("done", (), {"returncode": 0, "stdout": "", "stderr": ""}))
    assert _lib.build() == _lib.LIB_PATH
    assert "all" in seen[0] and "host" in seen[0]


def test_objects_follow_the_flags_they_are_built_with():
    """a Makefile with other flags (the one that left packed fp32 arithmetic out) makes every object anew, not those alone whose sources changed"""
    sources = [f for f in os.listdir(CSRC) if f.endswith((".hip", ".cpp")) and f != "host.cpp"]
    out = commands("-W", "Makefile")
    assert all(f" -c {f} " in out for f in sources) and "-packed-fp32-ops" in out, out
    assert "host.cpp" in commands("-W", "Makefile", "host")


def test_loads_in_inline_asm_wait_in_their_own_block():
    """the compiler takes an asm's outputs as written where it stands: a load whose wait stands in a later statement can be copied, or its
    register given away, while it is in flight"""
    import re
    load = re.compile(r"\b(ds_read|ds_load|global_load|buffer_load|flat_load|scratch_load|s_load|s_buffer_load)\w*")
    seen = 0
    for name in sorted(os.listdir(CSRC)):
        if not name.endswith((".hip", ".h", ".cpp")):
            continue
        text = open(os.path.join(CSRC, name)).read()
        for m in re.finditer(r"\basm\s*(volatile)?\s*\(", text):
            strings = re.match(r'(\s*"(?:[^"\\]|\\.)*")+', text[m.end():])
            body = strings.group(0) if strings else ""
            if load.search(body):
                seen += 1
                assert "s_waitcnt" in body, (name, text.count("\n", 0, m.start()) + 1, body[:80])
    assert seen >= 4
