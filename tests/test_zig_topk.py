"""Static checks of zig/hip_topk.zig, which no compiler here reads: every entry point of include/zg_hip_topk.h is called once, with
an argument of the right kind for each of its parameters."""
import re
from pathlib import Path

from zigrad_amd._lib import TOPK_HEADER, parse_header

TEXT = (Path(__file__).resolve().parent.parent / "zig" / "hip_topk.zig").read_text()


def calls():
    for m in re.finditer(r"c\.(zg_hip_\w+)\(", TEXT):
        depth, start, args = 1, m.end(), []
        for i in range(m.end(), len(TEXT)):
            depth += (TEXT[i] == "(") - (TEXT[i] == ")")
            if depth == 0 or (depth == 1 and TEXT[i] == ","):
                args.append(TEXT[start:i].strip())
                start = i + 1
            if depth == 0:
                break
        yield m.group(1), args


def test_every_entry_point_is_called_once_with_arguments_of_its_parameters_kinds():
    source = re.sub(r"/\*.*?\*/", "", Path(TOPK_HEADER).read_text(), flags=re.S)
    declared = parse_header(TOPK_HEADER)
    seen = [(name, args) for name, args in calls() if name != "zg_hip_last_error"]
    assert sorted(n for n, _ in seen) == sorted(declared)
    for name, args in seen:
        types = [" ".join(p.split()) for p in re.search(name + r"\s*\((.*?)\)\s*;", source, re.S).group(1).split(",")]
        assert len(types) == len(args), name
        for t, a in zip(types, args):
            param = re.search(r"(\w+)$", t).group(1)
            if param == "ctx":
                assert a == "ctx(device)"
            elif "uint64_t *" in t:
                assert re.fullmatch(r"@ptrCast\((?:\w+\.)?(\w+)\.ptr\)", a).group(1) == param, (name, a)
            elif "*" in t:
                assert re.fullmatch(r"(?:optional(?:_out)?\()?(?:\w+\.)?(\w+)(?:\.ptr|\))", a).group(1) == param, (name, a)
            elif t.startswith("int "):
                assert re.fullmatch(r"@intFromBool\((?:\w+\.)?(\w+)\)", a).group(1) == param, (name, a)
            else:
                assert re.fullmatch(r"(?:\w+\.)?(\w+)", a).group(1) == (param if param != "n_entries" else "len"), (name, a)


def test_brackets_match():
    code = re.sub(r"//.*", "", TEXT)
    for a, b in ("()", "{}", "[]"):
        assert code.count(a) == code.count(b)
