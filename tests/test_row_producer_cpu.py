"""The K and V producer warps of the packed and tree attention kernel on the
host: their source block is cut out of row_attn.cuh and run by 32 threads
(row_producer_emu.cpp). Whatever wait gives up, every lane has to get out of
the block: a lane left behind in a warp-wide operation would keep its CTA on
the GPU for ever."""
import shutil
import subprocess
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent
SOURCE = HERE.parent / "kvm_b200" / "csrc" / "row_attn.cuh"


@pytest.fixture(scope="module")
def emu(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    text = SOURCE.read_text()
    head, tail = "if (warp == 10 || warp == 14) {\n", "    } else if (warp == 11) {\n"
    assert text.count(head) == 1 and text.count(tail) == 1, "the producers' block has moved"
    where = tmp_path_factory.mktemp("row_producer")
    block = text[text.index(head) + len(head):text.index(tail)]
    (where / "row_producer_block.inc").write_text(block)
    exe = where / "row_producer_emu"
    subprocess.run(["g++", "-std=c++20", "-O1", "-pthread", "-Wno-unknown-pragmas", "-I", where,
                    HERE / "row_producer_emu.cpp", "-o", exe], check=True)
    return exe


@pytest.mark.parametrize("tree", [0, 1])
@pytest.mark.parametrize("kv", [0, 1])
def test_every_lane_leaves_whichever_wait_gives_up(emu, tree, kv):
    for grants in (0, 1, 2, 3, 7, 19, 20, 21, 22, 23):     # 23 tiles: the last never gives up
        r = subprocess.run([emu, str(tree), str(kv), str(grants)], capture_output=True, text=True,
                           timeout=60)
        assert r.returncode == 0, (grants, r.stderr)
        assert r.stdout == f"{grants} tiles\n"
