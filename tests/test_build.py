"""The in-tree build: what is compiled again, and what a failure leaves.  Compilers are stand-ins that write files."""
import os

import pytest

from triton_op_b200 import build as b

CUDA = sorted(s for s in b.SOURCES if s != b.CALLS_SOURCE)


@pytest.fixture
def compiled(tmp_path, monkeypatch):
    """The sources compiled by each build, in a library folder of the test's own; ["fail"] names those that fail."""
    lib = tmp_path / "lib"
    monkeypatch.setattr(b, "LIB_DIR", str(lib))
    monkeypatch.setattr(b, "LIB_PATH", str(lib / "lib.so"))
    monkeypatch.setattr(b, "CALLS_PATH", str(lib / "calls.so"))
    monkeypatch.setattr(b, "_nvcc", lambda: "/opt/cuda/bin/nvcc")
    log = {"now": [], "linked": 0, "fail": ()}

    class Job:
        def __init__(self, command, **kw):
            source = os.path.basename(next(c for c in command if c.endswith((".cu", ".cpp"))))
            if command[0] == "g++" and log.get("no g++"):
                raise FileNotFoundError("g++")
            log["now"].append(source)
            self.returncode = 1 if source in log["fail"] else 0
            with open(command[command.index("-o") + 1], "w") as f:
                f.write(" ".join(command))

        def communicate(self):
            return "said the compiler", None

    def link(command, **kw):
        log["linked"] += 1
        with open(command[command.index("-o") + 1], "w") as f:
            f.write("".join(open(o).read() for o in command if o.endswith(".o")))
        return type("Done", (), dict(returncode=0, stdout="", stderr=""))

    monkeypatch.setattr(b.subprocess, "Popen", Job)
    monkeypatch.setattr(b.subprocess, "run", link)

    def build(**kw):
        log["now"].clear()
        b.build(**kw)
        return sorted(log["now"])
    build.log = log
    return build


def test_nothing_is_built_twice(compiled):
    assert compiled() == sorted(b.SOURCES)
    assert compiled() == [] and not b.needs_build()
    os.utime(b.LIB_PATH, (1, 1))                                     # a library older than its sources
    assert b.needs_build()


def test_objects_of_another_kind_are_not_linked(compiled):
    """A library with clock stamps, then an ordinary one: every object is compiled again."""
    compiled(trace=True)
    assert "PA_TRACE_BUILD" in open(b.LIB_PATH).read()
    assert b.needs_build() and not b.needs_build(trace=True)
    assert compiled() == CUDA
    assert "PA_TRACE_BUILD" not in open(b.LIB_PATH).read()
    assert not b.needs_build()


def test_another_torch_builds_the_host_calls_again(compiled, monkeypatch):
    import torch
    compiled()
    monkeypatch.setattr(torch, "__version__", torch.__version__ + ".other")
    assert b.needs_build()
    assert compiled() == [b.CALLS_SOURCE]
    assert not b.needs_build()


@pytest.mark.parametrize("why", ["no g++", "fail"])
def test_the_library_is_built_where_the_host_calls_are_not(compiled, why):
    compiled.log[why] = True if why == "no g++" else (b.CALLS_SOURCE,)
    with pytest.raises(RuntimeError, match=b.CALLS_SOURCE):
        compiled()
    assert compiled.log["linked"] == 1 and os.path.exists(b.LIB_PATH) and not os.path.exists(b.CALLS_PATH)
    compiled.log[why] = ()
    assert compiled() == [b.CALLS_SOURCE]                            # the objects that are there stay


def test_a_failed_object_leaves_no_library_of_old_ones(compiled):
    compiled()
    compiled.log["fail"] = (CUDA[0],)
    with pytest.raises(RuntimeError, match=CUDA[0]):
        compiled(trace=True)
    assert b.needs_build() and b.needs_build(trace=True)
    compiled.log["fail"] = ()
    compiled()
    assert "PA_TRACE_BUILD" not in open(b.LIB_PATH).read()
