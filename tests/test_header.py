"""The C header against the sources: every entry point is defined with the
return and argument types it is declared with (the sources do not include the
header, so the compiler does not say)."""

import re
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def prototypes(text, end):
    """{name: (return type, argument types)} of what `end` closes."""
    text = re.sub(r"/\*.*?\*/", " ", text, flags=re.S)
    text = re.sub(r"//[^\n]*", "", text)
    found = {}
    for kind, name, args in re.findall(
            r"^(?:extern \"C\" )?((?:const )?(?:int|int64_t|char|void)\*?) (qx_\w+)\(([^()]*)\)\s*" + end, text, re.M):
        kinds = [re.sub(r"\s*\b\w+$", "", " ".join(a.split())).replace(" *", "*")
                 for a in args.split(",")] if args.strip() not in ("", "void") else []
        found[name] = (kind, tuple(kinds))
    return found


def test_every_entry_point_is_defined_as_it_is_declared():
    declared = prototypes((ROOT / "include" / "quail_mi355x.h").read_text(), ";")
    defined = {}
    for path in sorted((ROOT / "quail_amd" / "csrc").glob("*.*")):
        defined.update(prototypes(path.read_text(), r"\{"))
    assert len(declared) > 50
    assert set(declared) == {n for n in defined if n in declared}
    assert {n: (declared[n], defined[n]) for n in declared if declared[n] != defined[n]} == {}
