"""Kernels of headers that several HIP objects of the library share have a name, a launch stub and a registration of their own in
each: with one name for all of them the linker keeps one object's stub, which then launches for the others, too, and an
object built from another state of the header gets arguments that it does not expect."""
import re
import subprocess

CALL = r"\b%s\s*<"


def _kernels_of_several_objects():
    from camelid_amd import build
    text = {p.name: p.read_text() for p in [*build.CSRC.glob("*.h"), *build.CSRC.glob("*.hip")]}
    defined = {}
    for name, t in text.items():
        for m in re.finditer(r"__global__\s+(?:__launch_bounds__\s*\((?:[^()]|\([^()]*\))*\)\s*)?void\s+(k_\w+)\s*\(", t):
            defined[m.group(1)] = name

    def reached(name, seen):
        if name in text and name not in seen:
            seen.add(name)
            for other in re.findall(r'#include "(\w+\.h)"', text[name]):
                reached(other, seen)
        return seen

    users = {}
    for src in build.HIP_SOURCES:
        files = reached(src, set())
        for kernel, home in defined.items():
            if home in files and any(re.search(CALL % kernel, text[f]) for f in files):
                users.setdefault(kernel, set()).add(src)
    assert len(defined) > 50 and "k_pa_join" in defined
    return {k: u for k, u in users.items() if len(u) > 1}


def test_shared_kernels_are_each_objects_own(native):
    from camelid_amd import _native
    shared = _kernels_of_several_objects()
    assert shared.get("k_pa_join") == {"serving.hip", "serving8.hip"}
    symbols = subprocess.run(["nm", "-C", str(_native.LIB_PATH)], capture_output=True, text=True, check=True).stdout
    for kernel, sources in shared.items():
        kinds = re.findall(r"(\w) (?:void )?cm::(?:__device_stub__)?%s\b" % kernel, symbols)
        assert len(kinds) >= 2 * len(sources) and all(k.islower() for k in kinds), (kernel, set(kinds))
