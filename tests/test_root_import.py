"""The package is found from the repository's root alone, without PYTHONPATH, and is the one that lies there."""

import os
import subprocess
import sys

from conftest import PKG, REPO


def test_import_from_the_root():
    env = {k: v for k, v in os.environ.items() if k != "PYTHONPATH"}
    code = ("import ssd, ssd._lib, ssd.engine.scoring as s; from ssd.ops import token_logprobs_ws_bytes; "
            "print(ssd.__version__, s.__file__, ssd._lib.LIB_PATH, sep='\\n')")
    out = subprocess.run([sys.executable, "-c", code], cwd=REPO, env=env, capture_output=True, text=True, check=True).stdout.split()
    import ssd

    assert out == [ssd.__version__, os.path.join(PKG, "ssd", "engine", "scoring.py"), os.path.join(PKG, "ssd", "libssd_mi355x.so")]
    assert os.path.dirname(ssd.__path__[0]) == PKG
