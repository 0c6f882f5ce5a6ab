"""Rules that the kernels' sources keep and that no run shows reliably when broken."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "metallora_b200" / "csrc"


def _kernels():
    """(file, name, signature, body) of every kernel, comments taken out."""
    found = []
    for path in sorted(CSRC.glob("*.cu")):
        text = re.sub(r"//[^\n]*", "", path.read_text())
        for m in re.finditer(r"__global__", text):
            start = text.index("{", m.end())
            depth, end = 0, start
            while True:
                depth += {"{": 1, "}": -1}.get(text[end], 0)
                end += 1
                if depth == 0:
                    break
            head = text[m.end():start]
            name = re.search(r"(\w+)\s*\(\s*(?:const|void|uint|int|float|T |O |\))", head.split(")", 1)[1]
                             if "__launch_bounds__" in head else head)
            found.append((path.name, name.group(1) if name else head, head, text[start:end]))
    return found


KERNELS = _kernels()


def test_kernels_are_found():
    names = {k[1] for k in KERNELS}
    assert {"mx_prep_kernel", "lora_bwd_kernel", "mx_quantize_blocks_kernel",
            "mx_dequantize_blocks_kernel", "mx_skinny_kernel", "mx_wgrad_kernel"} <= names, names


def test_programmatic_dependents_load_coherently():
    """A kernel that starts while its input is still being written may not read it
    through the read-only path, which wants it unchanged for the grid's whole life."""
    seen = 0
    for file, name, head, body in KERNELS:
        if "grid_wait()" not in body:
            continue
        seen += 1
        text = re.sub(r"//[^\n]*", "", (CSRC / file).read_text())
        assert "__ldg(" not in body and "ld.global.nc" not in text, (file, name)
        assert "__restrict__" not in head, (file, name)
    assert seen >= 5


def test_stage_release_depends_on_the_loads():
    """The quantising warps hand a stage back by an arrive that hangs on what they
    loaded.  Compared with a constant, the condition (a maximum's bits are never all
    ones) could be folded away, and with it the order."""
    body = next(k[3] for k in KERNELS if k[1] == "mx_prep_kernel")
    arrive = re.search(r"if \(__reduce_max_sync\([^;]*?\) != ([\w.]+)[^;]*\)\s*mbar_arrive\(", body)
    assert arrive and arrive.group(1).startswith("p."), arrive


def test_first_kernels_wait_in_every_role():
    """The kernels that follow whatever ran before them wait for it in every role of
    their warps, ahead of that role's first bounded wait: one that went on would count
    a long predecessor against the limit."""
    roles = {"mx_prep_kernel": ("if (warp == 0) {", "else if (warp == 1) {", "else if (has_work) {"),
             "lora_bwd_kernel": ("if (warp == 0) {", "else if (warp == 1) {", "if (epi && has_work) {")}
    for name, starts in roles.items():
        body = next(k[3] for k in KERNELS if k[1] == name)
        for start in starts:
            role = body[body.index(start):]
            assert "grid_wait();" in role[:role.index("mbar_wait(")], (name, start)


def test_dependents_start_after_the_wait():
    """A kernel lets the next one start after its own wait: the next one reads ahead of
    its wait what is older than this kernel."""
    for file, name, head, body in KERNELS:
        if "grid_wait()" in body and "launch_dependents()" in body:
            assert body.index("grid_wait()") < body.index("launch_dependents()"), (file, name)
