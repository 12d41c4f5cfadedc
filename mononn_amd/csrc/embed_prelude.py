"""Build step: wrap the device headers into C++ string constants (device/prelude_text.h) so the host compiler can hand
them to hipRTC as includes.  Arguments: destination, then constant name=source file pairs."""
import sys

delim = "MONONN_PRELUDE"
with open(sys.argv[1], "w") as f:
    f.write("// generated by embed_prelude.py - do not edit\n#pragma once\n")
    f.write("namespace mononn { namespace device {\n")
    for arg in sys.argv[2:]:
        name, src = arg.split("=")
        text = open(src).read()
        assert ")" + delim not in text
        chunks = [text[i:i + 12000] for i in range(0, len(text), 12000)]   # stay under compilers' literal limits
        f.write(f"static const char {name}[] =\n")
        for c in chunks:
            f.write('R"' + delim + "(" + c + ")" + delim + '"\n')
        f.write(";\n")
    f.write("} }\n")
