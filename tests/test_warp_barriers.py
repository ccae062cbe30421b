"""CPU check of the sources: barriers that whole warps have to enter together (PTX .aligned; bar.sync is one) stand
only in the helpers of csrc/gx_device.cuh, which bring a warp's lanes together first. A warp whose lanes arrive
apart, after a loop or branch that depends on the lane, would be counted twice or hang."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "gyro-dx_b200" / "csrc"
BARRIER = re.compile(r'"[^"]*\b(?:barrier\.cluster\.\S*aligned|bar\.sync|barrier\.sync\.aligned)')


def test_aligned_barriers_are_entered_by_whole_warps():
    found = 0
    for path in sorted(CSRC.glob("*.cu*")):
        lines = path.read_text().splitlines()
        for i, line in enumerate(lines):
            if not BARRIER.search(line):
                continue
            assert path.name == "gx_device.cuh", f"{path.name}:{i + 1}"
            assert "__syncwarp();" in lines[i - 1], f"{path.name}:{i + 1}"
            found += 1
    assert found >= 4
