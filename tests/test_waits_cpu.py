"""The kernels' bounded waits: which of them a caller's budget bounds."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "cpu_ops_b200" / "csrc"


def calls(text, name):
    """Argument lists of the calls of `name`, split at their outer commas."""
    for at in re.finditer(re.escape(name) + r"\(", text):
        depth, args, start = 1, [], at.end()
        for i in range(at.end(), len(text)):
            depth += {"(": 1, ")": -1}.get(text[i], 0)
            if depth == 0 or (depth == 1 and text[i] == ","):
                args.append(text[start:i].strip())
                start = i + 1
            if depth == 0:
                break
        yield args


def test_waits_for_copies_under_way_do_not_go_by_the_callers_budget():
    """A CTA that gives up waits for what it has issued before it leaves.  With the budget that a caller may set to a
    microsecond that wait would end before a copy lands; such waits are mbar_drain's.  All others end
    with their CTA's abort flag too."""
    seen, drains = 0, 0
    for path in sorted(CSRC.glob("*")):
        text = path.read_text()
        drains += sum(1 for _ in calls(text, "mbar_drain"))
        for args in calls(text, "mbar_wait_bounded"):
            if args[0].startswith("uint32_t") or args[-1] == "kDrainLimitNs":
                continue   # the function itself, and mbar_drain
            seen += 1
            assert args[2] in ("abort_flag", "&abort_flag"), (path.name, args)
    assert seen > 20 and drains > 8
