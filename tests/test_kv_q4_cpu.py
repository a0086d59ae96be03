"""The cache in 4 bits on the host: where a page's codes and scales lie, and how a step's attention is cut into CTAs."""
import os
import subprocess

import numpy as np
import pytest

from densecore_b200 import build as B


def _program(tmp_path, text):
    src, exe = tmp_path / "p.cu", str(tmp_path / "p")
    src.write_text('#include <stdio.h>\n#include <stdlib.h>\n#include "dc_q4.h"\n' + text)
    subprocess.check_call([B.nvcc(), "-std=c++17", "--expt-relaxed-constexpr", "-arch=sm_100", "-I", B.CSRC, "-I", os.path.join(B.ROOT, "include"), str(src), "-o", exe])
    return exe


def test_every_code_has_a_place_of_its_own_and_no_byte_two_tokens(tmp_path):
    """Nibbles of keys and values over the whole record, against the lanes' view of mma.m16n8k16: lane (h, t) takes tokens h, h + 8 as key columns and
    tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9 as value rows."""
    exe = _program(tmp_path, r"""
template <int HD> void all() {
    using R = dc_q4_rec<HD>;
    for (int tok = 0; tok < 16; ++tok)
        for (int d = 0; d < HD; ++d) {
            const int word = R::k_word(tok, (d & 7) >> 1, d >> 5), nib = ((d >> 3) & 3) + 4 * (d & 1);
            printf("%d %d %d %d %d %d\n", HD, tok, d, 2 * (word + nib / 2) + nib % 2, 2 * R::v_byte(tok, d & 7, d >> 4) + ((d >> 3) & 1), R::BYTES);
        }
}
int main() { all<64>(); all<128>(); }
""")
    a = np.array([[int(x) for x in line.split()] for line in subprocess.check_output([exe], text=True).splitlines()])
    for hd in (64, 128):
        r = a[a[:, 0] == hd]
        k, v = r[:, 3], r[:, 4]
        assert set(r[:, 5]) == {18 * hd}
        assert sorted(k) == list(range(16 * hd)) and sorted(v) == list(range(2 * 9 * hd, 2 * 9 * hd + 16 * hd))
        for place in (k, v):
            assert len({(p // 2, t) for p, t in zip(place, r[:, 1])}) == 8 * hd      # a byte, a token
        # lanes: 16 bytes of key codes a lane and half (HD 128), or both halves in one (HD 64)
        lane_k = (k // 2 % 512) // 16
        assert np.array_equal(lane_k, (r[:, 1] % 8) * 4 + (r[:, 2] % 8) // 2)
        lane_v = ((v // 2 - 9 * hd) % 512) // 16
        assert np.array_equal(lane_v, (r[:, 2] % 8) * 4 + (r[:, 1] % 8) // 2)


@pytest.mark.parametrize("G,n_kv", [(1, 1), (3, 2), (8, 4), (16, 1)])
def test_items_cover_every_page_once(tmp_path, G, n_kv):
    exe = _program(tmp_path, r"""
int main(int, char** v) {
    std::vector<dc_q4_entry> es = {{3, 0, 1, 0}, {0, 15, 1, 1}, {1, 16, 1, 2}, {2, 4095, 5, 3}, {5, 100000, 1, 8}, {4, 0, 700, 9}};
    std::vector<dc_q4_item> items;
    int tickets, ws;
    dc_q4_items(es, atoi(v[1]), atoi(v[2]), 148, &items, &tickets, &ws);
    printf("%d %d\n", tickets, ws);
    for (auto& i : items) printf("%d %d %d %d %d %d %d %d %d %d %d\n", i.seq, i.pos0, i.tok0, i.count, i.tile, i.page0, i.page1, i.split, i.n_splits, i.ws, i.ticket);
}
""")
    lines = [[int(x) for x in line.split()] for line in subprocess.check_output([exe, str(G), str(n_kv)], text=True).splitlines()]
    tickets, ws = lines[0]
    tiles, taken, named = {}, set(), {}
    for seq, pos0, tok0, count, tile, p0, p1, split, n, at, ticket in lines[1:]:
        assert p0 < p1
        tiles.setdefault((seq, pos0, count, tile), []).append((p0, p1, split, n))
        if n > 1:
            assert 0 <= at + split < ws and (at + split) not in taken and 0 <= ticket < tickets
            taken.add(at + split)
            assert named.setdefault(ticket, (seq, tile)) == (seq, tile)
    assert len(taken) == ws and len(named) == tickets
    want = {(3, 0, 1): 1, (0, 15, 1): 1, (1, 16, 1): 1, (2, 4095, 5): 5, (5, 100000, 1): 1, (4, 0, 700): 700}
    for (seq, pos0, count), rows in want.items():
        for tile in range(-(-rows * G // 8)):
            got = sorted(tiles.pop((seq, pos0, count, tile)))
            last = pos0 + min(count - 1, (8 * tile + 7) // G)
            assert got[0][0] == 0 and got[-1][1] == last // 16 + 1
            assert all(x[1] == y[0] for x, y in zip(got, got[1:])) and [x[2] for x in got] == list(range(len(got))) and {x[3] for x in got} == {len(got)}
    assert not tiles


@pytest.mark.parametrize("G,n_kv", [(1, 1), (3, 2), (8, 4), (16, 1)])
def test_prompt_tiles_cover_every_row_and_key_once(tmp_path, G, n_kv):
    exe = _program(tmp_path, r"""
int main(int, char** v) {
    std::vector<dc_q4_entry> es = {{3, 0, 64, 0}, {0, 15, 2000, 64}, {1, 100000, 300, 2064}, {2, 63, 1, 2364}};
    if (atoi(v[3])) es.resize(1), es.push_back({1, 100000, 300, 64});
    std::vector<dc_q4_tile> tiles;
    int ws;
    dc_q4_tiles(es, atoi(v[1]), atoi(v[2]), 148, &tiles, &ws);
    printf("%d\n", ws);
    for (auto& t : tiles) printf("%d %d %d %d %d %d %d %d %d %d\n", t.seq, t.pos0, t.tok0, t.count, t.row0, t.tile0, t.tile1, t.split, t.n_splits, t.ws);
}
""")
    for short in (0, 1):
        lines = [[int(x) for x in line.split()] for line in subprocess.check_output([exe, str(G), str(n_kv), str(short)], text=True).splitlines()]
        ws, taken, got = lines[0][0], set(), {}
        for seq, pos0, tok0, count, row0, t0, t1, split, n, at in lines[1:]:
            assert t0 < t1
            got.setdefault((seq, pos0, count, row0), []).append((t0, t1, split, n))
            if n > 1:
                assert 0 <= at + split < ws and (at + split) not in taken
                taken.add(at + split)
        assert len(taken) == ws
        sizes = [line[6] - line[5] for line in lines[1:]]
        assert sizes == sorted(sizes, reverse=True)
        for seq, pos0, count in ([(3, 0, 64), (0, 15, 2000), (1, 100000, 300), (2, 63, 1)] if not short else [(3, 0, 64), (1, 100000, 300)]):
            for row0 in range(0, count * G, 256):
                parts = sorted(got.pop((seq, pos0, count, row0)))
                last = pos0 + (min(row0 + 256, count * G) - 1) // G
                assert parts[0][0] == 0 and parts[-1][1] == last // 64 + 1 and all(x[1] == y[0] for x, y in zip(parts, parts[1:]))
                assert [x[2] for x in parts] == list(range(len(parts))) and {x[3] for x in parts} == {len(parts)}
        assert not got


def test_the_prompt_kernel_is_built_without_spills(tmp_path):
    """It loads from tensor memory: the launcher refuses a build that spills."""
    import re
    cmd = [B.nvcc(), "-Xptxas", "-v", *B.NVCC_FLAGS, "-I", os.path.join(B.ROOT, "include"), "-c", os.path.join(B.CSRC, "attn_q4_prompt.cu"), "-o", str(tmp_path / "o.o")]
    out = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, check=True).stdout
    seen = [body for name, body in re.findall(r"Compiling entry function '(\w+)'(.*?)(?=Compiling entry|\Z)", out, re.S) if "k_q4_prompt" in name]
    assert len(seen) == 2 and all("0 bytes stack frame, 0 bytes spill stores, 0 bytes spill loads" in body for body in seen)


def test_null_arguments_are_refused():
    import ctypes as C
    from densecore_b200 import _lib
    lib = _lib.lib()
    out = C.c_void_p()
    assert lib.dc_b200_kv_create_q4(None, 1, 1, 1, 128, 0, 1, 1, 1, C.byref(out)) == -1
    assert lib.dc_b200_kv_batch(None, 0, None, None, None) == -1
    assert lib.dc_b200_kv_q4_write_dev(None, None, 0, None, None, 0, None, None) == -1
    assert lib.dc_b200_flash_attn_q4_dev(None, None, 0, None, 0, None, None, 0, 1.0, None, 0, None, None) == -1
    assert lib.dc_b200_flash_attn_q4(None, None, 0, None, None, None, 1.0, None) == -1
    assert lib.dc_b200_kv_q4_read_block(None, 0, 0, None, None) == -1
