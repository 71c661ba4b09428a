"""The paged calls' checks and plans on the host: the entry points' own source
with the launchers replaced by ones that print what they are asked for and
refuse what the kernels would (tests/paged_host.cc); and u15h_rope_freqs."""
import math
import pathlib
import random
import re
import shutil
import subprocess

import pytest

import paged_ref as ref
import u15h

REPO = pathlib.Path(__file__).resolve().parent.parent
CSRC = REPO / "vpipe-sensenova-u1.5_amd" / "csrc"
ROCM_INCLUDE = pathlib.Path("/opt/rocm/include")
SCRATCH = 32 << 20


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    if shutil.which("g++") is None or not ROCM_INCLUDE.exists():
        pytest.skip("g++ or the HIP headers not available")
    exe = tmp_path_factory.mktemp("paged") / "paged_host"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-D__HIP_PLATFORM_AMD__",
                    f"-I{ROCM_INCLUDE}", f"-I{REPO / 'include'}", f"-I{CSRC}",
                    str(REPO / "tests" / "paged_host.cc"), "-o", str(exe)], check=True,
                   timeout=300)

    def run(calls, cus=256, scratch=SCRATCH):
        out = subprocess.run([str(exe), str(cus), str(scratch)], input="\n".join(calls) + "\n",
                             capture_output=True, text=True, check=True, timeout=300).stdout
        lines = out.splitlines()
        assert len(lines) == len(calls)
        return [tuple(line.split(" ; ", 1)) for line in lines]
    return run


# ---- refusals: nothing is launched -------------------------------------------

ROPE = ["tokens=-1", "tokens=4194305", "heads=0", "heads=4097", "d=0", "d=513 width0=128",
        "spec=0", "pos=0", "pos=4098", "nparts=0", "nparts=4", "width0=0", "width0=3",
        "width0=130", "start0=-2 width0=4", "start0=126 width0=4", "axis0=3", "axis0=-1",
        "freq0=0", "freq0=4100", "rscale=inf", "rscale=nan", "x=0", "y=0", "x=4097", "y=8193",
        "x_tok=-8", "y_head=-1", "y_tok=64", "y_head=64", "y_tok=1000",
        "nparts=2 width0=64 start1=63 width1=4", "nparts=2 width0=64 start1=0 width1=4",
        "x_tok=2048", "x_tok=2e12"]
CACHE = ["kv=0", "d=48", "page=8", "page=48", "page=2097152", "heads=0", "pages=-1",
         "pages=134217728", "page_stride=16", "page_stride=16388", "page_stride=2e10",
         "kp=0", "vp=0", "kp=4104", "vp=4098"]
APPEND = CACHE + ["tokens=-1", "tokens=4194305", "slot=0", "slot=4097", "k=0", "v=0", "k=4104",
                  "k_stride=8", "v_stride=1020", "q=0", "q_out=0", "spec=0", "hq=0", "hq=5000",
                  "q_stride=8", "q_out_stride=4100", "pos=0", "nparts=4", "q_stride=8192",
                  "width0=256"]
ATTN = CACHE + ["batches=0", "hq=0", "hq=12", "hq=8192", "batch=-1", "batch=65537 tokens=65537",
                "tokens=-1", "max_q=-1", "max_kv=-1", "max_kv=536870912",
                "prefix_len=536870912", "prefix_len=-1", "table_stride=-1", "scale=-1",
                "scale=nan", "scale=inf", "scale=1e-20", "scale=1e20", "q_start=0 tokens=2",
                "kv_len=0", "kv_len=4098", "table=0", "table=4097", "q_start=4098",
                "prefix_len=5 prefix_table=0", "prefix_table=4099", "q=0", "out=0", "q=4104",
                "q_stride=8", "out_stride=4100", "hq=4096 tokens=1048576",
                "batch=65536 tokens=65536 heads=32"]


@pytest.mark.parametrize("name,bad", [("rope", ROPE), ("append", APPEND), ("attn", ATTN)])
def test_refusals_launch_nothing(host, name, bad):
    fine = {"rope": "rope", "append": "append", "attn": "attn"}[name]
    assert host([fine])[0][1] == "ok"
    for case, (launch, st) in zip(bad, host([f"{name} {b}" for b in bad])):
        assert launch == "-" and st != "ok" and st.startswith(
            {"rope": "rope", "append": "paged_append", "attn": "paged_attention"}[name]), \
            (case, launch, st)
    assert host([f"{name} ctx=0"]) == [("-", "refused")]


def test_empty_calls_launch_nothing(host):
    calls = ["rope tokens=0", "append tokens=0", "append tokens=0 slot=0 k=0 v=0 q=0 q_out=0",
             "attn batch=0 tokens=0", "attn tokens=0 max_q=0", "attn max_q=0",
             "attn batch=0 tokens=3"]
    assert host(calls) == [("-", "ok")] * len(calls)


def test_calls_that_are_allowed(host):
    calls = ["rope x=4098 y=4098 x_tok=1025 y_tok=1025 x_head=128 y_head=128", "rope x=4100",
             "rope y=8192 x_tok=0 x_head=0", "rope y_tok=128 y_head=640 x_tok=128 x_head=640",
             "append q=0 q_out=0 hq=0", "append q=0 q_out=0 hq=0 spec=0 pos=0",
             "append q=8192 q_out=8192", "attn kp=0 vp=0 pages=0", "attn table=0 max_kv=0",
             "attn table=0 table_stride=0", "attn q_start=0", "attn scale=0.5", "attn batch=65536"
             " tokens=65536"]
    for call, (launch, st) in zip(calls, host(calls)):
        assert st == "ok" and launch != "-", call
    assert "stride=0" in host(["attn table=0 max_kv=0"])[0][0]      # nothing to look up


def test_access_width_and_parts(host):
    """Columns an access: 8 where parts, strides and addresses allow, 2, 1; parts
    in order, their pairs numbered through."""
    want = {"rope": 8, "rope x=4100": 2, "rope y=4098": 1, "rope x_tok=1026 y_tok=1026": 2,
            "rope width0=56": 2, "rope width0=54": 1, "rope width0=54 neighbours=1": 2,
            "rope width0=56 neighbours=1": 8, "rope start0=4 width0=64": 2,
            "rope start0=1 width0=64": 1, "rope d=12 width0=8 heads=2": 2,
            "rope d=33 width0=32 heads=2": 1, "append start0=2 width0=64": 2}
    for call, (launch, st) in zip(want, host(list(want))):
        assert st == "ok" and f"vec={want[call]} " in launch, (call, launch)
    parts = "nparts=3 start0=96 width0=32 axis0=2 start1=0 width1=64 start2=64 width2=32 axis2=1"
    launch, _ = host([f"rope {parts}"])[0]
    assert launch.endswith("pairs=64 heads=8+0+0 sign=1 slots=0 parts 0:64:0:0 64:32:32:5 "
                           "96:32:48:10")
    assert "sign=-1" in host(["rope inverse=1"])[0][0]


# ---- plans ------------------------------------------------------------------------

@pytest.mark.parametrize("name", list(ref.PLANS))
def test_every_way_to_cut_a_call_has_a_gpu_case(host, name):
    """The cases that test_gpu_paged.py runs are cut as they say."""
    launch, st = host([ref.plan_call(name)])[0]
    assert st == "ok" and re.search(ref.PLANS[name][-1], launch), launch


@pytest.mark.parametrize("cus,scratch", [(256, SCRATCH), (256, 0), (64, SCRATCH), (1, 1 << 20)])
def test_every_batch_has_a_plan(host, cus, scratch):
    """Random batches: parts fit the scratch, chunks cover the keys (the host
    program's launcher checks), and without scratch nothing is cut."""
    rng = random.Random(cus + scratch)
    calls = []
    for _ in range(3000):
        batch = int(2 ** rng.uniform(0, 12))
        max_q = 1 if rng.random() < 0.5 else int(2 ** rng.uniform(0, 11))
        hkv = rng.choice([1, 2, 8, 32])
        calls.append(
            f"attn batch={batch} "
            f"tokens={min(max(batch, int(batch * max_q * rng.random())), 1 << 22)} "
            f"max_q={max_q} max_kv={int(2 ** rng.uniform(0, 20))} "
            f"prefix_len={rng.choice([0, int(2 ** rng.uniform(0, 20))])} heads={hkv} "
            f"hq={hkv * rng.choice([1, 4, 7, 80])} d={rng.choice([32, 64, 128])}"
            + rng.choice(["", " q_start=0"]))
    kinds = set()
    for call, (launch, st) in zip(calls, host(calls, cus, scratch)):
        assert st == "ok" or "too many" in st, (call, st)
        if st == "ok":
            kinds.add(re.search(r"(none|stream|tile)", launch).group(1))
            assert scratch or "parts=1 " in launch, (call, launch)
    assert kinds == ({"none", "stream", "tile"} if scratch else {"none"})


def test_counters_are_cleared_before_they_count(host):
    """By the first call that counts; a captured one leaves that to the next."""
    join, other = "attn batch=1 heads=2 hq=8 max_kv=1800", "attn batch=3"
    got = [launch.split(" parts")[0] for launch, _ in host(
        [other, join + " capturing=1", join + " capturing=1", join, join, join + " capturing=1"])]
    assert got == ["attn", "clear attn", "clear attn", "clear attn", "attn", "attn"]


# ---- frequencies ------------------------------------------------------------------

def test_rope_freqs():
    """Against the formulas; the two scalings by turns keep the fastest pairs and
    divide the slowest by the factor."""
    for width in (2, 64, 128):
        f, s = u15h.rope_freqs(width, 5e6)
        assert s == 1.0 and f.shape == (width // 2,)
        assert all(math.isclose(float(v), 5e6 ** (-2 * i / width), rel_tol=1e-14)
                   for i, v in enumerate(f))
        g, _ = u15h.rope_freqs(width, 5e6, "linear", factor=4.0)
        assert bool(((g * 4 - f).abs() <= 1e-15 * f).all())
    g, _ = u15h.rope_freqs(64, 1e4, "ntk", factor=8.0)
    # the slowest pair turns as if positions were squeezed by the factor
    f, _ = u15h.rope_freqs(64, 1e4)
    assert math.isclose(float(g[-1]), float(f[-1]) / 8.0, rel_tol=1e-12) and float(g[0]) == 1.0
    for kind in ("yarn", "bands"):
        g, s = u15h.rope_freqs(128, 1e4, kind, factor=8.0, trained=4096)
        f, _ = u15h.rope_freqs(128, 1e4)
        ratio = (g / f).tolist()
        assert ratio[0] == 1.0 and math.isclose(ratio[-1], 1 / 8, rel_tol=1e-14)
        assert all(a >= b - 1e-15 for a, b in zip(ratio, ratio[1:]))
        assert math.isclose(s, 0.1 * math.log(8.0) + 1.0 if kind == "yarn" else 1.0, rel_tol=1e-6)
        turns = [4096 * float(v) / (2 * math.pi) for v in f]
        slow, fast = 1.0, 32.0 if kind == "yarn" else 4.0
        if kind == "bands":
            for r, t in zip(ratio, turns):
                keep = min(max((t - slow) / (fast - slow), 0.0), 1.0)
                assert math.isclose(r, keep + (1 - keep) / 8, rel_tol=1e-12)
        else:
            lo = max(math.floor(128 * math.log(4096 / (fast * 2 * math.pi)) / (2 * math.log(1e4))), 0)
            hi = min(math.ceil(128 * math.log(4096 / (slow * 2 * math.pi)) / (2 * math.log(1e4))), 127)
            for i, r in enumerate(ratio):
                out = min(max((i - lo) / (hi - lo), 0.0), 1.0)
                assert math.isclose(r, 1 - out + out / 8, rel_tol=1e-12)


@pytest.mark.parametrize("kw", [dict(width=0), dict(width=3), dict(width=514), dict(theta=1.0),
                                dict(theta=math.inf), dict(theta=math.nan),
                                dict(scaling="linear", factor=0.5),
                                dict(scaling="ntk", factor=math.inf),
                                dict(scaling="yarn", factor=2.0, trained=0),
                                dict(scaling="bands", factor=2.0, trained=8, slow=4.0, fast=4.0),
                                dict(scaling="yarn", factor=2.0, trained=8, slow=0.0)])
def test_rope_freqs_refusals(kw):
    with pytest.raises(u15h.U15hError):
        u15h.rope_freqs(**{"width": 64, "theta": 1e4, **kw})


def test_rope_freqs_unknown_scaling():
    with pytest.raises(ValueError):
        u15h.rope_freqs(64, 1e4, "dynamic")
