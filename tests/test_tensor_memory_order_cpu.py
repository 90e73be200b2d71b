"""The order of two steps in every kernel that takes tensor memory, read from the sources.

A kernel that has let its successor start can find that successor's tensor memory on its own SM, held until the
successor's wait for this very kernel ends.  An allocation made after that moment may then never return.  So a
kernel allocates first, meets at a CTA barrier, and only then lets the next one start, unless its shared memory
leaves no room on the SM for any other kernel that holds tensor memory (`fills_sm`).
"""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "strata-masonry_b200" / "csrc"


def _code(path):
    text = re.sub(r"/\*.*?\*/", "", path.read_text(), flags=re.S)
    return re.sub(r"//[^\n]*", "", text)


def _bodies(text):
    for m in re.finditer(r"\)\s*\{", text):
        depth, i = 0, m.end() - 1
        while True:
            depth += {"{": 1, "}": -1}.get(text[i], 0)
            if depth == 0:
                break
            i += 1
        yield text[m.end():i]


def _holders():
    """(file, its code, kernel body) of everything that allocates and frees tensor memory."""
    found = []
    for path in sorted(CSRC.glob("*.cu")):
        code = _code(path)
        found += [(path.name, code, body) for body in _bodies(code) if "tmem_alloc<" in body and "tmem_dealloc<" in body]
    return found


HOLDERS = _holders()


def test_every_gemm_source_is_seen():
    names = [h[0] for h in HOLDERS]
    assert set(names) == {p.name for p in CSRC.glob("gemm_*.cu")}
    assert names.count("gemm_nvfp4_decode.cu") == 2


@pytest.mark.parametrize("name,code,body", HOLDERS, ids=[f"{i}-{h[0]}" for i, h in enumerate(HOLDERS)])
def test_successors_start_after_the_allocation(name, code, body):
    barrier = body.index("__syncthreads", body.index("tmem_alloc<"))
    early, late = [], []
    for line in re.finditer(r"[^\n]*griddep_launch_dependents\s*\([^\n]*", body):
        (late if line.start() > barrier else early).append(line.group().strip())
    assert len(early) <= 1 and len(late) <= 1 and early + late
    if early and not early[0].startswith("if (fills_sm(C::kTotal))"):
        assert "static_assert(fills_sm(kTotal)" in code, f"{name}: the next kernel may start before the allocation"
    elif early:
        assert late and late[0].startswith("if (!fills_sm(C::kTotal))"), name


def test_no_two_holders_fit_where_one_fills_the_sm():
    """The least shared memory of a holder is asserted beside every budget that is not asserted to fill the SM."""
    common = _code(CSRC / "gemm_common.cuh")
    least = int(re.search(r"kHolderShared = (\d+) \* 1024", common).group(1)) * 1024
    whole = int(re.search(r"kSmShared = (\d+) \* 1024", common).group(1)) * 1024
    assert whole == 228 * 1024 and 0 < least < whole // 2      # 227 KB for a CTA, 1 KB set aside for each
    for name in {h[0] for h in HOLDERS}:
        code = _code(CSRC / name)
        assert "static_assert(fills_sm(kTotal)" in code or ">= kHolderShared" in code, name
