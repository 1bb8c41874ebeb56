"""The scripts that build the library's sources by themselves know all of them, and build them as the library is built."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def text(*path):
    return open(os.path.join(ROOT, *path)).read()


def test_scripts_build_what_the_library_is_built_of():
    make = text("cleanba_amd", "csrc", "Makefile")
    sources = {f[:-4] for f in re.search(r"^SRCS = (.*)$", make, re.M)[1].split()}
    assert "tokens" in sources and sources == {f[:-4] for f in os.listdir(os.path.join(ROOT, "cleanba_amd", "csrc")) if f.endswith(".hip")}
    variants = text("tools", "variants.sh")
    link = next(line for line in variants.splitlines() if "-shared" in line and "-o ../abl_" in line)
    assert {os.path.basename(o)[:-2] for o in re.findall(r"\S+\.o\b", link)} == sources   # (a library that lacks one does not load)
    check = text("tools", "check_no_dispatch_ptr.sh")
    lists = re.findall(r"^for f in (.*); do$", check, re.M)
    assert len(lists) == 2 and all(set(names.split()) == sources for names in lists)
    for script in (variants, check):
        assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in script and "-ffp-contract=off" in script
