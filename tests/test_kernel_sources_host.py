"""CPU: what has to stand in a kernel's source, for faults that no run may be made to show."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "oxicuda_b200" / "csrc"


def _code(name):
    text = (CSRC / name).read_text()
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


def test_every_thread_of_the_few_token_product_waits_for_the_previous_kernel():
    """All threads, in front of the roles: a thread that stores or begins a bounded wait before the previous kernel of the stream has ended
    could overwrite what that kernel still reads, or count its time."""
    code = _code("gemm_fp8_block128_few.cu")
    body = code[code.index("gemm_block128_few_kernel("): code.index("int32_t launch(")]
    at = re.search(r'\n  asm volatile\("griddepcontrol\.wait;" ::: "memory"\);', body)       # two spaces: no branch around it
    assert at, "no wait that every thread executes"
    roles = body.index("if (warp == 0)")
    assert at.start() < roles and not re.search(r"\b(mbar_wait|warp_wait)\(", body[: at.start()])
    limit = re.search(r"kWaitLimitNs = (\d+)ull", code)
    assert int(limit.group(1)) <= 2_000_000_000                     # a failure is seen within seconds
