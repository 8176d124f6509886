"""The build on a tree that holds no built file yet."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_module_builder_loads_without_the_module_it_builds(tmp_path):
    # a copy of the sources as they come from history: flash_ck/ without its compiled module
    (tmp_path / "flash_ck").mkdir()
    for name in ("__init__.py", "build.py"):
        (tmp_path / "flash_ck" / name).write_text(open(os.path.join(ROOT, "flash_ck", name)).read())
    (tmp_path / "__graft_entry__.py").write_text(open(os.path.join(ROOT, "__graft_entry__.py")).read())
    r = subprocess.run([sys.executable, "-c", "import __graft_entry__ as g; m = g.module_builder(); assert callable(m.build); print(m.target())"],
                       cwd=tmp_path, env={k: v for k, v in os.environ.items() if k != "PYTHONPATH"}, stdout=subprocess.PIPE,
                       stderr=subprocess.STDOUT, text=True)
    assert r.returncode == 0, r.stdout
    assert r.stdout.strip().startswith(str(tmp_path))
