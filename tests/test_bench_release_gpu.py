"""bench.py: the legs behind the headline load tables of their own, so the headline's have to be gone by then — its server, its caches and
its sessions, none of them kept by a name that a loop left behind (with the default 133 GB of tables both would not fit the host)."""
import json
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


@pytest.mark.gpu
@pytest.mark.parametrize("args", [("--gpus", "1", "--no-triton-leg", "--no-wide-leg", "--no-direct-leg", "--no-c3-leg"),
                                  ("--gpus", "1", "--mode", "async", "--no-triton-leg", "--no-wide-leg", "--no-direct-leg", "--no-c3-leg"),
                                  ("--gpus", "2", "--no-extra-legs")])
def test_the_headline_is_released_before_the_legs_behind_it(tmp_path, args):
    r = subprocess.run([sys.executable, str(ROOT / "bench.py"), "--rows", "100000", "--batch", "2048", "--steps", "2", "--warmup", "1", "--blocks", "2",
                        "--no-cpu-baseline", "--no-sharded-leg", *args], capture_output=True, text=True, timeout=100, cwd=tmp_path)
    assert r.returncode == 0, r.stderr[-3000:]
    full = json.loads((Path(tmp_path) / "bench_extra.json").read_text())
    assert full["headline_objects_left"] == 0, r.stderr[-2000:]
    assert full["parity_vs_oracle_bit_exact"] is not False
