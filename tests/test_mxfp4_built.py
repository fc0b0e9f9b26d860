"""The built MXFP4 product kernels, as the code objects in the library hold them: what their hand-counted waits rest on."""
import os
import re
import struct
import subprocess

import pytest

import llama_box_amd as L
from test_host_and_abi import built_kernels

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


def code_objects(data):
    """the gfx950 code objects in a library's bytes"""
    magic, at = b"__CLANG_OFFLOAD_BUNDLE__", -1
    while (at := data.find(magic, at + 1)) >= 0:
        n, p = struct.unpack_from("<Q", data, at + 24)[0], at + 32
        for _ in range(n):
            off, size, chars = struct.unpack_from("<QQQ", data, p)
            if size and b"gfx950" in data[p + 24:p + 24 + chars]:
                yield data[at + off:at + off + size]
            p += 24 + chars


def waits(lines):
    """[(n, requests)] of every wait in front of a barrier, vmcnt(n), that stands behind DMA into LDS of the same straight run of code: n, and the vector memory requests between the last DMA and it"""
    found, behind = [], None
    for line, after in zip(lines, list(lines[1:]) + [""]):
        word = line.split()[0] if line.split() else ""
        if "_load_lds_" in word:
            behind = 0
        elif re.match(r"(s_cbranch|s_branch|s_setpc|s_endpgm)", word):
            behind = None
        elif behind is not None and re.match(r"(global|buffer|flat|scratch)_(load|store|atomic)", word):
            behind += 1
        elif behind is not None and word == "s_waitcnt" and after.split()[:1] == ["s_barrier"] and (m := re.search(r"vmcnt\((\d+)\)", line)):
            found.append((int(m[1]), behind))
    return found


def test_reading_of_a_listing():
    ok = ["global_load_lds_dwordx4 v1, s[2:3]", "buffer_load_dwordx4 v[2:5], v1, s[0:3], 0 offen", "buffer_load_dwordx2 v[2:3], v1, s[0:3], 0 offen", "v_mov_b32 v1, v2", "s_waitcnt vmcnt(2) lgkmcnt(0)", "s_barrier"]
    assert waits(ok) == [(2, 2)]
    assert waits([ok[1], ok[0]] + ok[2:]) == [(2, 1)]  # (a request that has moved in front: the wait does not cover the DMA)
    assert waits(ok[:3] + ["s_cbranch_scc1 12"] + ok[3:]) == [] and waits(ok[:-1] + ["v_mov_b32 v1, v2"]) == []


@pytest.fixture(scope="module")
def listing(built, tmp_path_factory):
    """{symbol: instructions} of the kernels of the file that holds the MXFP4 products"""
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    with open(L.BACKEND_SO, "rb") as f:
        elfs = [e for e in code_objects(f.read()) if b"k_mx_wide" in e]
    assert len(elfs) == 1
    path = tmp_path_factory.mktemp("mx") / "mx.elf"
    path.write_bytes(elfs[0])
    text = subprocess.run([OBJDUMP, "-d", "--mcpu=gfx950", str(path)], capture_output=True, text=True, check=True).stdout
    return {m[1]: m[2].splitlines() for m in re.finditer(r"<(\w+)>:\n(.*?)(?=\n\n|\Z)", text, re.S)}


def test_no_scratch(built):
    """no MXFP4 kernel spills: a launch with a scratch frame pays for it at every dispatch, and the frame is read back ahead of the first weights"""
    kernels = {name: m for name, m in built_kernels().items() if re.search(r"k_mx_|k_add_id", name)}
    assert len(kernels) > 20 and not {name: m[".private_segment_fixed_size"] for name, m in kernels.items() if m[".private_segment_fixed_size"]}


def test_results_stay_in_reach_of_their_reader(listing):
    """no store of a product goes past the caches, from where the next node reads it"""
    stores = [ln for name, lines in listing.items() if "k_mx_" in name for ln in lines if re.search(r"\b(global|buffer|flat)_store", ln)]
    assert stores and not [ln for ln in stores if re.search(r"\b(nt|sc1)\b", ln)]


def test_stage_waits_cover_the_dma(listing):
    """k_mx_wide waits for a stage's DMA with vmcnt(n), n digit requests behind the last DMA: requests complete in order, so at least n of them have to lie there in every build of it"""
    kernels = {name: lines for name, lines in listing.items() if "k_mx_wide" in name}
    assert len(kernels) == 6  # two, four and eight row tiles, of one matrix and of experts
    for name, lines in kernels.items():
        counted = [(n, behind) for n, behind in waits(lines) if n > 0]
        # (two loops a height, for the even and the odd quarters of a row; the launch of eight row tiles of one matrix holds the lower tiles', too)
        assert len(counted) == (6 if "ILb0ELi8E" in name else 2), (name, counted)
        assert all(behind >= n for n, behind in counted), (name, counted)
