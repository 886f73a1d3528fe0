"""The package from a checkout's root, with nothing but the root on the path."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PACKAGE = os.path.join(ROOT, "flash-evict-prefill_b200")


def python(code, *path):
    env = {k: v for k, v in os.environ.items() if k != "PYTHONPATH"}
    lines = [f"import sys; sys.path[:] = {list(path)!r} + [p for p in sys.path if p not in ('', {ROOT!r}, {PACKAGE!r})]", code]
    r = subprocess.run([sys.executable, "-c", "\n".join(lines)], cwd=ROOT, env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    return r.stdout.split()


@pytest.mark.parametrize("path", [(ROOT,), (PACKAGE,), (ROOT, PACKAGE), (PACKAGE, ROOT)])
def test_one_package_whatever_is_on_the_path(path):
    got = python("from flash_evict.decode import KVCache\n"
                 "import flash_evict, flash_evict._lib, flash_evict.decode\n"
                 "assert flash_evict.decode.KVCache is KVCache and flash_evict is sys.modules['flash_evict']\n"
                 "assert flash_evict.evict and 'evict' in flash_evict.__all__ and flash_evict.__doc__\n"
                 "print(flash_evict.__file__, flash_evict.decode.__file__, flash_evict._lib.__file__)", *path)
    want = os.path.join(PACKAGE, "flash_evict")
    assert got == [os.path.join(want, f) for f in ("__init__.py", "decode.py", "_lib.py")]
