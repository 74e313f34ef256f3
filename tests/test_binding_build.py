"""The compiled binding of the serving-step operators: what it was built for, and when it is built."""
import subprocess
import sys

from fgw_b200 import _native, build


def test_a_binding_of_another_header_is_refused(tmp_path):
    """A binding left over from an older header would hand over structures of another layout."""
    header = (build.INCLUDE / "fgw_mha.h").read_text()
    line = f"#define FGW_MHA_ABI_VERSION {_native.ABI_VERSION}\n"
    assert line in header
    include, lib = tmp_path / "include", tmp_path / "lib"
    include.mkdir()
    lib.mkdir()
    (include / "fgw_mha.h").write_text(header.replace(line, "#define FGW_MHA_ABI_VERSION 4\n"))
    (lib / build.LIB.name).symlink_to(build.LIB)
    made = subprocess.run([*build.binding_command(lib / build.BINDING.name, include), "-O0"], capture_output=True, text=True)
    assert made.returncode == 0, made.stderr
    # in a process of its own: a process has one module of the name
    load = ("import pathlib, sys; from fgw_b200 import _native; _native.LIB_PATH = pathlib.Path(sys.argv[1])\n"
            "try: _native.torch_binding()\n"
            "except _native.NativeLibraryError as error: print('refused:', error)")
    ran = subprocess.run([sys.executable, "-c", load, str(lib / build.LIB.name)], capture_output=True, text=True,
                         cwd=build.ROOT)
    assert ran.returncode == 0 and ran.stdout.startswith("refused:") and "rebuild" in ran.stdout, ran
    _native.torch_binding()  # the tree's own is good


def binding_builds(monkeypatch):
    """How often build() makes the binding from here on (the compiler is not run)."""
    made = []
    monkeypatch.setattr(build, "_build_binding", lambda: made.append(1))
    return made


def test_the_binding_is_built_again_for_another_torch_or_python(tmp_path, monkeypatch):
    made = binding_builds(monkeypatch)
    monkeypatch.setattr(build, "BINDING_STAMP", tmp_path / "stamp")
    build.build()
    assert len(made) == 1  # nothing says what the present one was built with
    build.build()
    assert len(made) == 1
    monkeypatch.setattr(build, "_version", lambda package: "0.0+other")
    build.build()
    assert len(made) == 2
    build.build()
    assert len(made) == 2
    monkeypatch.setattr(build.sys, "version", "another interpreter")
    build.build()
    assert len(made) == 3


def test_the_library_builds_without_torch(tmp_path):
    """Users of the C ABI need no torch: the library is built, the binding left out."""
    run = ("import pathlib, sys; sys.modules['torch'] = None; from fgw_b200 import build\n"
           "build.BINDING = pathlib.Path(sys.argv[1]); build.BINDING_STAMP = build.BINDING.with_suffix('.stamp')\n"
           "print(build.build() == build.LIB, build.BINDING.exists())")
    ran = subprocess.run([sys.executable, "-c", run, str(tmp_path / "fgw_torch.so")], capture_output=True, text=True,
                         cwd=build.ROOT)
    assert ran.returncode == 0, ran.stderr
    assert ran.stdout.splitlines()[-1] == "True False" and "without torch" in ran.stdout
