"""The Julia wrapper, read as text (nothing executes it here): names that older versions of Julia lack are looked up only
where they exist, since a name in a method's signature is looked up when the module is loaded."""
import os
import re

import lvd_pg_b200

WRAPPER = os.path.join(os.path.dirname(lvd_pg_b200.__file__), "julia", "PCB200.jl")


def test_bfloat16_is_named_only_where_julia_has_it():
    with open(WRAPPER) as f:
        text = "".join(line for line in f if not line.lstrip().startswith("#"))
    guarded = re.compile(r"^@static if isdefined\(Core, :BFloat16\)\n(.*?)^else\n.*?^end\n", re.S | re.M)
    inside = "".join(m.group(1) for m in guarded.finditer(text))
    assert text.count("Core.BFloat16") == inside.count("Core.BFloat16") > 0
    assert "const WideScale = Core.BFloat16" in inside and "const WideScale = Float16" in text
