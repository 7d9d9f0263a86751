"""The kernel and the pieces that a step of drafted tokens takes, by the rules of esda_tree_forms.h on the host."""
import os
import subprocess

import pytest

from _tree_forms import STEPS

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def form_of(tmp_path_factory):
    exe = tmp_path_factory.mktemp("forms") / "tree_forms_check"
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I", os.path.join(ROOT, "include"),
                        "-I", os.path.join(ROOT, "apertura_amd", "csrc"), os.path.join(ROOT, "tests", "tree_forms_check.cpp"), "-o", str(exe)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr

    def forms(steps):
        """Lines of (batch, nodes, Hq, Hkv, D, K = V, window, room, split_rows)."""
        r = subprocess.run([str(exe)], input="\n".join(" ".join(str(int(x)) for x in s) for s in steps), capture_output=True, text=True)
        assert r.returncode == 0, r.stderr
        return r.stdout.splitlines()

    return forms


def test_forms_of_the_steps_that_cover_them(form_of):
    lines = [(len(lengths), T, hq, hkv, D, shared, 0, room, split) for (D, hq, hkv, T, lengths, room, split), shared, _ in STEPS]
    assert form_of(lines) == [form for *_, form in STEPS]


def test_the_steps_cover_every_form():
    found = {(step[0], shared, form) for step, shared, form in STEPS}
    kernels = {128: ["run 16 4", "run 32 4", "tile 128 4"], 256: ["run 16 4", "tile 64 8", "tile 128 8"], 512: ["run 16 4", "tile 64 4", "tile 128 8"]}
    assert found == {(D, shared, f"{k} {n}") for D, ks in kernels.items() for k in ks for shared in (False, True) for n in ("one", "split")}


def test_forms_by_query_rows_and_room(form_of):
    """The rules' borders: query rows of a kv head, the room's 10 and 100 MB, and what the GPU holds at once."""
    def kind(B, T, hq, hkv, D, shared, room):
        return form_of([(B, T, hq, hkv, D, shared, 0, room, 2 ** 31 - 32)])[0].rsplit(" ", 1)[0]

    # D = 128: two heads, K and V: 1,024 bytes a row
    assert [kind(1, T, 4, 2, 128, 0, 9000) for T in (8, 9, 64)] == ["run 16 4"] * 3               # 16, 18, 128 rows, small
    assert [kind(1, T, 16, 2, 128, 0, 50000) for T in (2, 3, 8, 9)] == ["run 16 4", "run 32 4", "run 32 4", "tile 128 4"]
    assert [kind(1, T, 16, 2, 128, 0, 110000) for T in (2, 4, 5)] == ["run 16 4", "run 32 4", "tile 128 4"]
    assert [kind(B, 64, 32, 2, 128, 0, 100) for B in (1, 8, 9)] == ["run 32 4"] * 2 + ["tile 128 4"]  # 512 workgroups of 32 rows
    # D = 256: 2,048 bytes
    assert [kind(1, T, 16, 2, 256, 0, 50000) for T in (2, 3, 8, 9)] == ["run 16 4", "tile 64 8", "tile 64 8", "tile 128 8"]
    assert [kind(1, T, 16, 2, 256, 0, 20000) for T in (2, 3, 9, 64)] == ["run 16 4", "tile 64 8", "tile 64 8", "tile 64 8"]
    assert [kind(B, 64, 32, 2, 256, 0, 100) for B in (8, 9)] == ["tile 64 8", "tile 128 8"]
    # D = 512: 4,096 bytes, K = V 2,048
    assert [kind(1, T, 16, 2, 512, 1, 10000) for T in (2, 4, 5, 8, 9, 16, 17)] == ["run 16 4"] * 2 + ["tile 64 4"] * 4 + ["tile 128 8"]
    assert [kind(1, T, 16, 2, 512, 0, 10000) for T in (2, 3, 8, 9, 16, 17)] == ["run 16 4", "tile 128 8", "tile 128 8", "tile 64 4", "tile 64 4", "tile 128 8"]
    assert [kind(1, T, 16, 2, 512, 0, 100) for T in (3, 32, 33)] == ["run 16 4", "run 16 4", "tile 64 4"]
