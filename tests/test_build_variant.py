"""CPU: tools/build_variant.sh compiles a unit as the Makefile does (a compiler that writes its arguments down stands in)."""
import os
import shutil
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_a_variant_differs_in_its_flags_alone(tmp_path):
    stub, log = tmp_path / "hipcc", tmp_path / "log"
    stub.write_text(f'#!/bin/bash\necho "$@" >> {log}\n')
    stub.chmod(0o755)
    name = f"test_{os.getpid()}"
    try:
        env = dict(os.environ, HIPCC=str(stub))
        units = ["kernels_gated.hip", "kernels_attention.hip", "kernels_norm.hip"]
        subprocess.run(["bash", "tools/build_variant.sh", name, "-DONE -DTWO"] + units, cwd=ROOT, env=env, check=True,
                       stdout=subprocess.DEVNULL)
        made = subprocess.run(["make", "-C", "tsdiff_amd/csrc", "--no-print-directory", "-n", "-B", "../libtsdiff_hip.so"], cwd=ROOT,
                              env=env, check=True, capture_output=True, text=True).stdout.splitlines()
    finally:
        shutil.rmtree(os.path.join(ROOT, "tools", "bin", f"obj_{name}"), ignore_errors=True)
    lines = log.read_text().splitlines()
    for u in units:
        obj = u.replace(".hip", ".o")
        want, = [m for m in made if f" -c {u} " in m]
        got, = [line for line in lines if f" -c {u} " in line]
        flags = want.split(" -o ")[0].split(" ", 1)[1]
        assert got == f"{flags} -DONE -DTWO -o {ROOT}/tools/bin/obj_{name}/{obj}"
        assert ("-amdgpu-mfma-vgpr-form" in got) == (u != "kernels_norm.hip")
    link, = [line for line in lines if "-shared" in line]
    assert all(f"/obj_{name}/{u[:-4]}.o" in link for u in units) and " api.o " in link
