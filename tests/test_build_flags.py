"""Every source that may hold kernels is compiled without packed float32."""
import os
import subprocess

from crowdllama_amd.ops import build


def test_no_kernel_with_packed_float32(monkeypatch, tmp_path):
    commands = []

    class Done:
        returncode = 0

        def __init__(self, cmd, **kw):
            commands.append(cmd)

        def communicate(self):
            return "", ""

    monkeypatch.setattr(subprocess, "Popen", Done)
    monkeypatch.setattr(subprocess, "run", Done)
    build.build(verbose=False, force=True)
    compiled = {os.path.basename(c[c.index("-c") + 1]): " ".join(c)
                for c in commands if "-c" in c}
    assert set(compiled) == set(build.SOURCES)
    flag = "-Xclang -target-feature -Xclang -packed-fp32-ops"
    for name in build.SOURCES:
        with open(os.path.join(build.CSRC, name)) as f:
            if "__global__" in f.read():
                assert flag in compiled[name], name
