"""The dense operators' host code and index arithmetic, replayed without a GPU by two programs that compile the sources
themselves: tests/cpp/dense_calls_test.cpp (every call's launches, workspace and planes) and tests/cpp/dense_tiles_test.cpp
(where a tile's values lie in memory and LDS)."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "silentotithrandousha_amd", "csrc")


def build(folder, name, *sources):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    out = str(folder / name)
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    os.path.join(ROOT, "tests", "cpp", name + ".cpp"), *(os.path.join(CSRC, s) for s in sources), "-o", out], check=True)
    return out


@pytest.fixture(scope="module")
def calls(tmp_path_factory):
    return build(tmp_path_factory.mktemp("calls"), "dense_calls_test", "dense_api.cpp", "dense_plan.cpp")


@pytest.fixture(scope="module")
def tiles(tmp_path_factory):
    return build(tmp_path_factory.mktemp("tiles"), "dense_tiles_test")


def replay(exe, lines, *mode):
    """(exit code, {call: its forms}, the last line) of lines as dense_calls_test.cpp describes them."""
    r = subprocess.run([exe, *(mode or ("calls",))], input="\n".join(lines), capture_output=True, text=True, timeout=100)
    out = r.stdout.splitlines()
    return r.returncode, dict(line.split(" : ") if " : " in line else (line, "") for line in out if " :" in line), out[-1]


# every kind of call, of one token, few, many, more than one piece; padded and odd sizes
CALLS = [f"{op} {T} {H} {X} {dtype}{tail}" for dtype in (0, 1) for T, H, X in ((1, 32, 8), (5, 96, 504), (21, 64, 1000), (22, 64, 1000),
         (333, 2048, 1536), (4096, 2880, 2880), (8197, 64, 4096), (20000, 160, 2056))
         for op, tail in (("loss", ""), ("lossgrad", " 1 1"), ("lossgrad", " 1 0"), ("lossgrad", " 0 1"), ("ffn", " 0"), ("ffn", " 1"),
                          *(("ffngrad", f" {kept} {mask}") for kept in (0, 1) for mask in (31, 1, 2, 4, 8, 16, 14, 27)))]
CALLS += [f"loss{g} {T} {H} {V} {dtype}{' 1 1' * bool(g)}" for g in ("", "grad") for dtype in (0, 1)
          for T, H, V in ((1, 2880, 201088), (16389, 32, 4097), (8200, 32, 33000), (8193, 64, 11001), (3, 32, 1), (2048, 2880, 201088))]


def test_calls_stay_in_their_buffers(calls):
    rc, got, last = replay(calls, CALLS)
    assert rc == 0 and last == "faults 0" and len(got) == len(set(CALLS))


# the largest vocabularies that the head of a card holds
WIDE = [f"loss {T} {H} {V} {dtype}" for dtype in (0, 1) for T in (1, 3, 16, 40, 300, 16384, 40000) for H, V in ((32, 2**25), (64, 2**28))]
WIDE += [f"lossgrad {T} {H} {V} 1 {dx} {dw}" for T in (1, 16, 40) for H, V in ((32, 2**28), (64, 2**28), (2880, 10**6)) for dx, dw in ((1, 1), (1, 0), (0, 1))]


def test_wide_heads(calls):
    """Grids of less than 2^32 threads, statistics of a bounded size (8.6 GB: 256 tokens of 2^28 rows)."""
    rc, got, last = replay(calls, WIDE, "calls", str(9 * 10**9))
    assert rc == 0 and last == "faults 0" and len(got) == len(WIDE)


def test_drawn_calls_stay_in_their_buffers(calls):
    r = subprocess.run([calls, "draw", "30000", "5"], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.splitlines()[-1] == "faults 0"


@pytest.mark.parametrize("mistake", ["slot", "behind", "short"])
def test_a_planted_mistake_in_a_call_is_found(calls, mistake):
    """Planes read from other slots, rows longer than they are, an allocation 4 KB short."""
    rc, _, last = replay(calls, CALLS, "plant", mistake)
    assert rc == 3 and last != "faults 0"


def test_products_that_do_not_fit_are_refused(calls):
    """Results leave in pieces of 16 bytes: rows of another length would be written behind."""
    r = subprocess.run([calls, "checks"], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout


def test_refusals(calls):
    r = subprocess.run([calls, "refusals"], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout


def test_workspace_growth(calls):
    """Lengths that rise by one do not allocate, and wait for the device, each time."""
    r = subprocess.run([calls, "growth"], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout


def test_tiles(tiles):
    r = subprocess.run([tiles], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout.splitlines()[-1]


@pytest.mark.parametrize("mistake,code", [("clamp", 3), ("pieces", 4)])
def test_a_planted_mistake_in_the_tiles_is_found(tiles, mistake, code):
    assert subprocess.run([tiles, mistake], capture_output=True, timeout=100).returncode == code


def plan_tiles():
    """(rows, columns, planes) of every tile shape of the plan."""
    text = open(os.path.join(CSRC, "dense_plan.hpp")).read()
    rows = [[int(float(v)) for v in m.split(",")] for m in re.findall(r"^  X\(([^)]*)\)", text, re.M)]
    return {(r[0], r[1], r[5]) for r in rows}


@pytest.fixture(scope="module")
def drawn(calls):
    """The forms that 200000 calls of 1 to 16384 tokens take."""
    r = subprocess.run([calls, "draw", "200000", "2"], capture_output=True, text=True, timeout=200)
    assert r.returncode == 0
    return {line.split(" : ")[0].strip() for line in r.stdout.splitlines() if " : " in line}


def test_every_tile_is_taken(drawn):
    """Each shape of the plan is some call's."""
    taken = set()
    for f in drawn:
        m = re.match(r"(?:store|gate|dgate|stats|dlogits)\.\w\w\.(\d+)x(\d+)(.*)", f)
        if m:
            taken.add((int(m[1]), int(m[2]), 3 if ".planes" in m[3] else 1))
    assert plan_tiles() == taken


def parameters(test):
    """The parameter sets of a test, as dicts."""
    sets = [{}]
    for m in test.pytestmark:
        if m.name == "parametrize":
            names = [n.strip() for n in m.args[0].split(",")]
            sets = [dict(s, **dict(zip(names, v if len(names) > 1 else (v,)))) for s in sets for v in m.args[1]]
    return sets


def lines_of(kind, T, H, X, dtype):
    """The calls that the GPU tests of a size make."""
    return {"loss": [f"loss {T} {H} {X} {dtype}", f"lossgrad {T} {H} {X} {dtype} 1 1"],
            "dx": [f"lossgrad {T} {H} {X} {dtype} 1 0"],
            "block": [f"ffn {T} {H} {X} {dtype} 0", f"ffngrad {T} {H} {X} {dtype} 0 31"],
            "kept": [f"ffn {T} {H} {X} {dtype} 1", f"ffngrad {T} {H} {X} {dtype} 1 31"]}[kind]


def sizes_run():
    from tests import dense_sizes as more
    from tests import test_gpu_dense as gpu
    kinds = [("loss", gpu.test_loss_and_gradient, "V"), ("loss", gpu.test_loss_tiles, "V"), ("block", gpu.test_block, "I"),
             ("block", gpu.test_block_tiles, "I"), ("kept", gpu.test_block_from_checkpoint, "I")]
    sizes = [(kind, p["T"], p["H"], p[x], p["dtype"]) for kind, test, x in kinds for p in parameters(test)]
    sizes += [("loss", p["T"], 32, p["V"], p["dtype"]) for p in parameters(gpu.test_loss_gradient_in_pieces)]
    for kind, sized in (("loss", more.LOSS), ("dx", more.LOSS_DX), ("block", more.BLOCK), ("kept", more.KEPT)):
        sizes += [(kind, *s) for s in sized]
    return sizes


def test_every_form_is_tested(calls, drawn):
    """The GPU tests run every form of launch that drawn calls take, against 64 bits."""
    rc, got, _ = replay(calls, [line for s in sizes_run() for line in lines_of(*s)])
    assert rc == 0
    assert drawn - set(" ".join(got.values()).split()) == set()
