"""Streams of the framework keep the default priority: a stream that waits for an event of one of another priority has not
come back on this part (docs/kernels.rst)."""
import ast
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def test_no_stream_asks_for_a_priority():
    found = []
    for path in [*ROOT.glob("*.py"), *ROOT.glob("p2pfl_amd/**/*.py"), *ROOT.glob("tools/**/*.py"), *ROOT.glob("perf/*.py"),
                 *ROOT.glob("examples/**/*.py")]:
        for node in ast.walk(ast.parse(path.read_text())):
            if isinstance(node, ast.Call) and any(k.arg in ("priority", "is_high_priority_stream") for k in node.keywords):
                found.append(f"{path.relative_to(ROOT)}:{node.lineno}")
    for path in [*ROOT.glob("p2pfl_amd/csrc/*"), *ROOT.glob("tools/**/*.hip")]:
        if path.is_file() and "StreamCreateWithPriority" in path.read_text(errors="ignore"):
            found.append(str(path.relative_to(ROOT)))
    assert not found
