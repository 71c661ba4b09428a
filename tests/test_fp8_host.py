"""The fp8 tier's checks and plans on the host: the entry points' own source
with the launchers replaced by ones that print what they are asked for and
refuse what the kernels would (tests/fp8_host.cc)."""
import pathlib
import random
import re
import shutil
import subprocess

import pytest

import fp8_ref as ref

REPO = pathlib.Path(__file__).resolve().parent.parent
CSRC = REPO / "vpipe-sensenova-u1.5_amd" / "csrc"
ROCM_INCLUDE = pathlib.Path("/opt/rocm/include")


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    if shutil.which("g++") is None or not ROCM_INCLUDE.exists():
        pytest.skip("g++ or the HIP headers not available")
    exe = tmp_path_factory.mktemp("fp8") / "fp8_host"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-D__HIP_PLATFORM_AMD__",
                    f"-I{ROCM_INCLUDE}", f"-I{REPO / 'include'}", f"-I{CSRC}",
                    str(REPO / "tests" / "fp8_host.cc"), "-o", str(exe)], check=True, timeout=300)

    def run(calls, cus=256):
        out = subprocess.run([str(exe), str(cus)], input="\n".join(calls) + "\n",
                             capture_output=True, text=True, check=True, timeout=300).stdout
        lines = out.splitlines()
        assert len(lines) == len(calls)
        return [tuple(line.split(" ; ", 1)) for line in lines]
    return run


def kernel_builds():
    """(family, rows, columns) of every product kernel, as built."""
    text = (CSRC / "u15h_fp8.hip").read_text()

    def rows(macro):
        block = re.search(rf"#define {macro}\(X\)((?:.*\\\n)*.*)", text).group(1)
        return [tuple(map(int, r.split(","))) for r in re.findall(r"X\(([\d, ]+)\)", block)]
    narrow = {("narrow", 16 * mt, 16 * fi) for mt, fi, *_ in rows("U15H_FP8_NARROW")}
    tiles = {("tiles", 16 * wm * fj, 16 * wn * fi)
             for wm, wn, fj, fi, *_ in rows("U15H_FP8_TILES")}
    return narrow | tiles


def parsed(launch):
    m = re.match(r"(narrow|tiles) (\d+)x(\d+) n=(\d+) tail=(\d+) shares=(\d+)", launch)
    return (m.group(1), *map(int, m.groups()[1:3])), *map(int, m.groups()[3:])


def random_gemms(n):
    rng = random.Random(7)
    calls = []
    for _ in range(n):
        mu, mg = rng.choice([(1, 0), (0, 1), (1, 1)])
        mu *= int(2 ** rng.uniform(0, 13))
        mg *= int(2 ** rng.uniform(0, 13))
        K = 16 * int(2 ** rng.uniform(0, 10))
        Ns = [8 * int(2 ** rng.uniform(0, 12)) for _ in range(rng.randint(1, 4))]
        calls.append(f"gemm {mu} {mg} {K} " + " ".join(map(str, Ns)))
    return calls


def test_every_build_is_reached_and_no_other(host):
    got = {parsed(launch)[0] for launch, st in host(random_gemms(4000)) if st == "ok"}
    assert got == kernel_builds()


@pytest.mark.parametrize("cus", [256, 208, 64, 1])
def test_every_product_has_a_plan(host, cus):
    """The launcher's own conditions and the workspace's size hold for each."""
    calls = random_gemms(1500)
    split = 0
    for call, (launch, st) in zip(calls, host(calls, cus)):
        assert st == "ok", (call, st)
        split += parsed(launch)[3] > 1
    assert split > 50 or cus == 1     # (one unit has no partial round of large tiles)


def test_the_largest_sizes(host):
    big = 1 << 22
    ok = [f"gemm {big} 0 131072 1048576", f"gemm 0 {big} 16 8", "gemm 1 0 131072 1048576",
          f"gemm 1 {big - 1} 128 1048576 1048576 8 8", f"rows {big} 131072",
          f"swiglu {big} 131072 1", f"norm {big} 0 16384 1 1 1", "blocks 1048576 131072"]
    for call, (launch, st) in zip(ok, host(ok)):
        assert st == "ok" and launch != "-", (call, st)
    no = [f"gemm {big} 1 128 8", "gemm 1 0 131088 8", "gemm 1 0 128 1048584",
          f"gemm 2147483647 2147483647 128 8", f"rows {big + 1} 16", "rows 1 131088",
          f"swiglu {big + 1} 16 0", f"norm 1 {big} 16 0 0 0", "norm 1 0 16400 0 0 0",
          "blocks 1048577 16", "blocks 1 131088"]
    for call, (launch, st) in zip(no, host(no)):
        assert launch == "-" and st.startswith("refused: "), (call, launch, st)


def test_the_larger_group_of_rows_comes_first(host):
    (launch, st), = host(["gemm 128 4096 4096 12288 12288"])
    assert st == "ok" and launch.endswith("rows 4096 4096 128 128")


def test_no_rows_no_launch(host):
    calls = ["gemm 0 0 256 8", "rows 0 256", "swiglu 0 256 0", "norm 0 0 256 1 1 0",
             "blocks 0 256"]
    assert host(calls) == [("-", "ok")] * len(calls)


@pytest.mark.parametrize("call", [
    "rows 4 0", "rows 4 8", "rows 4 -16", "rows -1 256", "swiglu 4 264 0", "blocks -8 256",
    "blocks 8 24", "norm 4 0 0 0 0 0", "norm -1 4 256 0 0 0", "gemm 1 0 120 8", "gemm 1 0 0 8",
    "gemm 1 0 128 4", "gemm 1 0 128 0", "gemm 1 0 128 8 12", "gemm -1 4 128 8", "gemm 4 -1 128 8",
    "gemm 4 0 128", "gemm 4 0 128 8 8 8 8 8"])
def test_sizes_refused(host, call):
    (launch, st), = host([call])
    assert launch == "-" and st.startswith("refused: ") and len(st) > 12, (launch, st)


@pytest.mark.parametrize("which", [
    "rows.x", "rows.q", "rows.s", "blocks.w", "blocks.q", "swiglu.up", "swiglu.h", "norm.delta",
    "norm.x_out", "norm.w_gen", "norm.eps", "norm.nan", "norm.y", "gemm.y", "gemm.wq_und",
    "gemm.sw_gen", "gemm.nproj", "gemm.proj", "gemm.sx", "context"])
def test_operands_refused(host, which):
    (launch, st), = host([f"bad {which}"])
    assert launch == "-" and st.startswith("refused: "), (launch, st)


def test_a_group_without_rows_needs_no_weights(host):
    (launch, st), = host(["bad none.gemm"])
    assert st == "ok" and launch != "-"


def test_the_sizes_that_stand_for_the_kernels(host):
    """Every build, and of the tiles each with and without shares of K and with
    one round of workgroups and more."""
    calls = ["gemm {} {} {} ".format(*size[:3]) + " ".join(map(str, size[3]))
             for size, *_ in ref.KINDS]
    seen = set()
    for (size, name, split, rounds), (launch, st) in zip(ref.KINDS, host(calls)):
        build, tiles, tail, shares = parsed(launch)
        slots = 512 if build[1] == 64 else 256
        assert st == "ok" and launch.startswith(name + " "), (size, launch)
        assert (shares > 1) == split and (name[0] == "n" or (tiles > slots) == rounds), launch
        seen.add(build)
    assert seen == kernel_builds()


def test_the_sizes_of_long_k(host):
    """The narrow ones pass 64 blocks of K a wave, the tiles have both whole
    rounds and shares."""
    calls = ["gemm {} {} {} ".format(*size[:3]) + " ".join(map(str, size[3]))
             for size, *_ in ref.LONG]
    for (size, name, split), (launch, st) in zip(ref.LONG, host(calls)):
        assert st == "ok" and launch.startswith(name + " "), (size, launch)
        assert (parsed(launch)[3] > 1) == split, (size, launch)
        assert ref.blocks(size[2]) > 4 * 64


def test_split_tails_are_partial_rounds(host):
    """What is split is what whole rounds of workgroups leave, a round being what
    the chip runs at once: on each unit as many tiles as its 160 KiB of LDS hold
    (NS stages of a float for each of 64 rows or columns and of 128 codes a row
    or column), at most eight multiplying waves."""
    text = (CSRC / "u15h_fp8.hip").read_text()
    rows = re.search(r"#define U15H_FP8_TILES\(X\)((?:.*\\\n)*.*)", text).group(1)
    per_cu = {}
    for row in re.findall(r"X\(([\d, ]+)\)", rows):
        wm, wn, fj, fi, _, ns, _ = map(int, row.split(","))
        bm, bn = 16 * wm * fj, 16 * wn * fi
        scales = -(-ns * 4 * (-(-bm // 64) * 64 + 64) // 1024) * 1024
        lds = scales + ns * 128 * (bm + bn)
        per_cu["tiles", bm, bn] = max(min(160 * 1024 // lds, 8 // (wm * wn)), 1)
    sized = ["gemm {} {} {} ".format(*size[:3]) + " ".join(map(str, size[3]))
             for size, *_ in ref.KINDS + ref.LONG]
    for cus in (256, 208):
        calls, seen = random_gemms(1500) + sized, set()
        for call, (launch, st) in zip(calls, host(calls, cus)):
            build, tiles, tail, shares = parsed(launch)
            if shares > 1:
                assert tail == tiles % (cus * per_cu[build]), (call, launch)
                seen.add(build)
        assert seen == set(per_cu) or cus != 256


def test_loaders_refuse_codes(tmp_path):
    """e4m3 tensors of a checkpoint are the caller's to load: the loaders of the
    other tiers say so and convert nothing."""
    import torch
    from safetensors.torch import save_file

    import u15h
    path = tmp_path / "w.safetensors"
    save_file({"p.weight": torch.zeros(8, 128, dtype=torch.float8_e4m3fn)}, str(path))
    with pytest.raises(u15h.U15hError) as err:
        u15h.load_matrix(None, path, "p", 128)
    assert err.value.status == u15h.EINVAL and "float8_e4m3fn" in str(err.value)
