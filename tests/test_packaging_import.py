"""A packed solution, unpacked somewhere else, is a package that imports: it holds every module that its own ``__init__`` needs."""
import os
import subprocess
import sys

from fused_moe_b200.packaging import pack_solution


def test_an_unpacked_solution_imports(tmp_path):
    for source in pack_solution.build_solution()["sources"]:
        path = tmp_path / source["path"]
        path.parent.mkdir(parents=True, exist_ok=True)
        path.write_text(source["content"])
    code = ("import binding, fused_moe_b200; from fused_moe_b200 import kernel; "
            "assert callable(kernel.custom_kernel); print(fused_moe_b200.__file__)")
    env = {k: v for k, v in os.environ.items() if k != "PYTHONPATH"}
    run = subprocess.run([sys.executable, "-c", code], cwd=tmp_path, env=env, capture_output=True, text=True)
    assert run.returncode == 0, run.stderr
    assert os.path.realpath(run.stdout.strip()).startswith(os.path.realpath(str(tmp_path)))
