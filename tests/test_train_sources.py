"""Rules of the kernels for training that a run cannot show without failing on the GPU, read from their sources."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "lightly_trian_quant_b200" / "csrc"
SOURCES = ("kf_norm.cu", "kf_rope.cu", "kf_attn_pack.cu", "kf_attn_pack_bwd.cu", "kf_attn.cuh")


def _code(name):
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


def test_read_only_loads_are_of_what_no_kernel_writes():
    """dependent launches may be resident while the kernel before them still writes its results, which the read-only path (__ldg, const __restrict__) does not allow for: it
    is for the plan's tables and the slopes, which the host makes."""
    for name in SOURCES:
        loads = re.findall(r"__ldg\(\s*([\w.]+)", _code(name))
        assert set(loads) <= {"a.slopes", "tiles"}, (name, loads)
        assert "__restrict__" not in _code(name), name


def test_register_splits_are_checked_against_the_build():
    """a kernel that hands registers from one role to another draws on those it was launched with; where a build gives it fewer, the role that asks for more waits without a limit:
    every such kernel's launch looks at what the build allocated first."""
    for path in sorted(CSRC.glob("*.cu")):
        code = _code(path.name)
        if "setmaxnreg_inc<" in code:
            assert "split_ready(" in code, path.name
            assert "cudaFuncAttributeMaxDynamicSharedMemorySize" not in code, path.name      # the look and this go together


def test_tensor_memory_is_given_back_before_a_cluster_waits():
    """a CTA that held tensor memory while it waits for the others of its cluster could stand against a cluster of another stream that does the same the other way round: the
    forward's parts give it back before they meet."""
    code = _code("kf_attn_pack.cu")
    assert code.count("tmem_dealloc(") == 1
    release = code[code.index("auto release = [&]()"):]
    assert "tmem_dealloc(" in release[:release.index("  };")] and "cluster_wait" not in release[:release.index("  };")]
    for at in (m.start() for m in re.finditer(r"cluster_wait\(\)|cluster_sync_all\(\)", code)):
        assert "release();" in code[:at][code[:at].rindex("if constexpr (SPLIT)"):], code[at - 200:at]


def test_rotary_positions_have_no_kernel_that_nothing_reaches():
    """the widest access is 16 bytes: eight 16-bit values, four of fp32"""
    from lightly_trian_quant_b200 import build

    build.build()
    (path,) = (build.CSRC / "build").glob("kf_rope.*.ptxas")
    kernels = set(re.findall(r"rope_axes_kernelI(\w+?)Li(\d)ELb(\d)E", path.read_text()))
    assert {v for t, v, _ in kernels if t.startswith("f")} == {"1", "2", "4"}
    assert {v for t, v, _ in kernels if not t.startswith("f")} == {"1", "2", "4", "8"}
    assert ("ff", "1", "1") not in kernels                       # pairs side by side need two values at once


def test_layer_norm_has_a_step_near_every_width():
    """values per lane are compiled in steps, and empty places of a step cost as much as full ones: no width pays for more than twice its own and two"""
    code = _code("kf_norm.cu")
    body = code[code.index("static int ln_by_width"):]
    body = body[:body.index("\n}\n")]
    body = body[body.index("const int n = (d + lanes - 1)"):]
    steps = [int(n) for n in re.findall(r"std::integral_constant<int, 1>\{\}, std::integral_constant<int, (\d+)>", body)]
    assert steps == sorted(steps) and [int(n) for n in re.findall(r"if \(n <= (\d+)\)", body)] == steps[:-1]
    for backward, warps in ((False, ((1024, 1), (2048, 2), (4096, 4), (8192, 8))), (True, ((512, 1), (1024, 2), (2048, 4), (8192, 8)))):
        for d in range(1, 8193):
            lanes = 32 * next(w for most, w in warps if d <= most)
            n = -(-d // lanes)
            step = next(s for s in steps if n <= s)
            assert step <= 2 * n + 2, (backward, d, n, step)
