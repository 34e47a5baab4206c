"""tools/build_variant.sh: a variant of any translation unit links with all the others and loads, an unknown unit is refused
(no GPU needed: hipcc cross-compiles gfx950)."""
import ctypes
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "mint_amd", "csrc")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


def _run(name, *args):
    return subprocess.run(["bash", os.path.join(ROOT, "tools", "build_variant.sh"), name] + list(args), capture_output=True,
                          text=True, timeout=1500)


@pytest.mark.parametrize("unit", ["probe", "qk_norm"])
def test_a_variant_loads_and_holds_its_unit(unit):
    if not shutil.which(HIPCC) and not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    name = "test_%s_%d" % (unit, os.getpid())
    path = os.path.join(ROOT, "tools", "bin", "libfact_%s.so" % name)
    mark = "variant_mark_%s" % name  # a flag that shows in the object: the source's file name, as the compiler notes it
    try:
        out = _run(name, unit, "-DFACT_VARIANT_TEST", "-ffile-prefix-map=%s=%s" % (CSRC, mark), "-g1")
        assert out.returncode == 0 and "built" in out.stdout, out.stderr[-3000:]
        with open(path, "rb") as f:
            assert mark.encode() in f.read(), "the unit that was compiled is not in the library"
        lib = ctypes.CDLL(path, mode=os.RTLD_NOW)
        assert lib.fact_abi_version() == 3
        for symbol in ("fact_attention", "fact_qk_norm_backward", "fact_debug_set_option"):
            assert hasattr(lib, symbol), symbol
    finally:
        if os.path.exists(path):
            os.remove(path)


def test_unknown_units_are_refused():
    name = "test_unknown_%d" % os.getpid()
    for args in (["no_such_unit"], ["engine_dbg"], []):
        out = _run(name, *args)
        assert out.returncode != 0 and "built" not in out.stdout
        assert not os.path.exists(os.path.join(ROOT, "tools", "bin", "libfact_%s.so" % name))


def test_every_source_is_a_unit():
    text = open(os.path.join(CSRC, "build.sh")).read()
    units = text.split('UNITS="', 1)[1].split('"', 1)[0].split() + ["engine", "probe"]
    assert sorted(units) == sorted(f[:-4] for f in os.listdir(CSRC) if f.endswith(".hip"))
