"""The sequence operators without a GPU: the C ABI of libtaco_sequence.so, what the host layer and the entry points refuse, the work lists, and the paged cache's index
arithmetic compiled for the host."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest
import torch

from taco_amd import _lib, sequence

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "taco_sequence.h")


@pytest.fixture(scope="module")
def lib():
    return sequence.load()


def test_header_library_and_binding_agree(lib):
    txt = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(taco_[a-z_]+)\s*\(", txt)))
    assert names == sorted(sequence.EXPORTS)
    for n in names:
        assert hasattr(lib, n)
    from taco_amd import build
    assert lib.taco_sequence_source_hash().decode() == build.sequence_hash() == build.embedded_hash(build.LIB_SEQ)
    syms = [line.split()[-1] for line in subprocess.check_output(["nm", "-D", "--defined-only", build.LIB_SEQ]).decode().splitlines()]
    assert sorted(s for s in syms if s.startswith("taco_")) == names
    assert "getenv" not in subprocess.check_output(["nm", "-D", build.LIB_SEQ]).decode()


def test_struct_layouts(tmp_path):
    structs = {"taco_seq_tensor": sequence.Tensor, "taco_attention_args": sequence.AttentionArgs, "taco_attention_step_args": sequence.AttentionStepArgs,
               "taco_linear_attention_args": sequence.LinearArgs, "taco_linear_attention_step_args": sequence.LinearStepArgs}
    lines = [f'printf("%zu\\n", sizeof({n}));' + "".join(f'printf("%zu\\n", offsetof({n}, {f[0]}));' for f in t._fields_) for n, t in structs.items()]
    src = tmp_path / "t.c"
    src.write_text('#include <stdio.h>\n#include "taco_sequence.h"\nint main(void) {' + "".join(lines) + "return 0; }")
    subprocess.check_call(["gcc", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), "-o", str(tmp_path / "t"), str(src)])
    got = [int(x) for x in subprocess.check_output([str(tmp_path / "t")]).split()]
    want = []
    for t in structs.values():
        want += [C.sizeof(t)] + [getattr(t, f[0]).offset for f in t._fields_]
    assert got == want


def tensor(p=1 << 20, ts=64, hs=32):
    return sequence.Tensor(p, ts, hs)


def attention_args(**kw):
    a = sequence.AttentionArgs(tensor(), tensor(), tensor(), tensor(), 1 << 20, 1 << 20, None, 1, 128, 0, 2, 2, 32, 0, 1, 1.0, tensor(), tensor(), tensor(), tensor(), 1 << 20, 1, None)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def step_args(**kw):
    a = sequence.AttentionStepArgs(tensor(), tensor(), tensor(), tensor(), 1 << 20, 1 << 20, 1024, 64, 32, 1024, 64, 32, 1 << 20, 4, 1 << 20, 2, 4, 8, 16, 2, 2, 32, 0, 1.0, None, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def linear_args(**kw):
    a = sequence.LinearArgs(tensor(), tensor(), tensor(), tensor(), 1 << 20, None, None, 1 << 20, 1 << 20, 2, 2, 2, 32, 0, 1.0, None, 0, tensor(), tensor(), tensor(), tensor(), None, None)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def linear_step_args(**kw):
    a = sequence.LinearStepArgs(tensor(), tensor(), tensor(), tensor(), 1 << 20, 1 << 20, None, 0, 2, 2, 32, 0, 1.0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


BAD_TENSORS = [tensor(p=None), tensor(p=(1 << 20) + 8), tensor(ts=30), tensor(ts=66), tensor(hs=-32), tensor(hs=34), tensor(ts=1 << 22)]


@pytest.mark.parametrize("name,make,bad", [
    ("taco_attention", attention_args, [dict(dim=12), dict(dim=0), dict(dim=136), dict(dtype=3), dict(heads=3), dict(kv_heads=0), dict(scale=0.0), dict(scale=float("nan")),
                                        dict(scale=float("inf")), dict(tile_rows=64), dict(whole=1), dict(n_tiles=-1), dict(n_tiles=1 << 30, heads=4), dict(lse=None), dict(tiles=None)]
     + [{f: t} for f in "qkvo" for t in BAD_TENSORS]),
    ("taco_attention_backward", attention_args, [dict(delta=None), dict(parts=0), dict(parts=3), dict(parts=2, kv_heads=1)] + [{f: t} for f in ("d_o", "d_q", "d_k", "d_v") for t in BAD_TENSORS]),
    ("taco_attention_step", step_args, [dict(rows=-1), dict(num_pages=0), dict(page_size=0), dict(table_width=0), dict(table=None), dict(lengths=None), dict(k_pages=None),
                                        dict(v_pages=(1 << 20) + 4), dict(k_page_stride=1022), dict(v_token_stride=-64), dict(scale=-1.0), dict(rows=1 << 30, heads=2),
                                        dict(k_new=tensor(p=None)), dict(v_new=tensor(p=None)), dict(q=tensor(hs=16))] + [{f: t} for f in ("q", "o") for t in BAD_TENSORS]),
    ("taco_linear_attention", linear_args, [dict(n_segments=1), dict(n_sequences=-1), dict(scale=0.0), dict(scale=float("inf")), dict(log_decay=None), dict(segments=None),
                                            dict(first_segment=None), dict(n_segments=90000, n_sequences=80000)] + [{f: t} for f in "qkvo" for t in BAD_TENSORS]),
    ("taco_linear_attention_backward", linear_args, [{f: t} for f in ("q", "d_o", "d_q", "d_k", "d_v") for t in BAD_TENSORS]),
    ("taco_linear_attention_step", linear_step_args, [dict(rows=-1), dict(scale=0.0), dict(state=None), dict(state=(1 << 20) + 4), dict(log_decay=None),
                                                      dict(reset=1 << 20, reset_bytes=2), dict(dim=10)] + [{f: t} for f in "qkvo" for t in BAD_TENSORS])])
def test_entry_points_refuse(lib, name, make, bad):
    """before any HIP call, with a message"""
    f = getattr(lib, name)
    assert f(None, None) == -1
    for kw in bad:
        assert f(C.byref(make(**kw)), None) == -1, kw
        assert lib.taco_sequence_last_error(), kw


def test_workspaces(lib):
    a = step_args(table_width=4096)
    need = lib.taco_attention_step_workspace_bytes(C.byref(a))
    assert need > 0 and lib.taco_attention_step(C.byref(a), None) == -3 and b"workspace" in lib.taco_sequence_last_error()
    a = step_args(table_width=4096, workspace=1 << 20, workspace_bytes=need - 1)
    assert lib.taco_attention_step(C.byref(a), None) == -3
    assert lib.taco_attention_step_workspace_bytes(C.byref(step_args())) == 0
    a = linear_args(n_segments=5)
    one, three = (lib.taco_linear_attention_workspace_bytes(C.byref(a), b) for b in (0, 1))
    assert one == 5 * 2 * 32 * 32 * 4 and three == 3 * one
    assert lib.taco_linear_attention(C.byref(a), None) == -3 and lib.taco_linear_attention_backward(C.byref(a), None) == -3
    # nothing to do is not an error, and launches nothing
    assert lib.taco_attention(C.byref(attention_args(n_tiles=0)), None) == 0
    assert lib.taco_attention_step(C.byref(step_args(rows=0)), None) == 0
    assert lib.taco_linear_attention(C.byref(linear_args(n_segments=0, n_sequences=0)), None) == 0
    assert lib.taco_linear_attention_step(C.byref(linear_step_args(rows=0)), None) == 0


def test_host_layer_refuses():
    z = torch.zeros(4, 2, 32)
    seqs = sequence.Packed([4], "cuda:0")
    with pytest.raises(_lib.TacoError, match="MI355X"):
        sequence.attention(z, z, z, seqs)
    with pytest.raises(_lib.TacoError, match="MI355X"):
        sequence.attention_step(z, z, z, z[None], z[None], torch.zeros(4, 1, dtype=torch.int32), torch.zeros(4, dtype=torch.int32))
    with pytest.raises(_lib.TacoError, match="MI355X"):
        sequence.linear_attention(z, z, z, torch.zeros(2), seqs)
    with pytest.raises(_lib.TacoError, match="MI355X"):
        sequence.linear_attention_step(z, z, z, torch.zeros(2), torch.zeros(4, 2, 32, 32))
    with pytest.raises(_lib.TacoError, match="MI355X"):
        sequence.Packed([4], "cpu")
    for lens in ([-1], [1.5], [[1, 2]], [2 ** 31]):
        with pytest.raises(ValueError):
            sequence.Packed(lens, "cuda:0")


class Fake:
    """what the checks look at of a tensor on a HIP device (no such device here)"""

    def __init__(self, shape, dtype=torch.float32, device="cuda:0", grad=False):
        self.t = torch.empty(shape, dtype=dtype, device="meta")
        self.device, self.dtype, self.shape, self.requires_grad = torch.device(device), dtype, self.t.shape, grad

    def dim(self):
        return self.t.dim()

    def __getattr__(self, name):
        return getattr(self.t, name)

    def data_ptr(self):
        return 1 << 20


def test_host_layer_refuses_shapes_and_types():
    F, s = Fake, sequence
    seqs = s.Packed([3, 1], "cuda:0")
    q, k = F((4, 4, 32)), F((4, 2, 32))
    for args in [(F((4, 32)), k, k), (q, F((5, 2, 32)), F((5, 2, 32))), (q, F((4, 3, 32)), F((4, 3, 32))), (q, k, F((4, 1, 32))), (q, F((4, 2, 40)), F((4, 2, 40))),
                 (q, F((4, 2, 32), torch.float16), k), (F((3, 4, 32)), F((3, 2, 32)), F((3, 2, 32))), (F((4, 4, 32), device="cuda:1"), F((4, 2, 32), device="cuda:1"), F((4, 2, 32), device="cuda:1"))]:
        with pytest.raises(ValueError):
            s.attention(*args, seqs)
    with pytest.raises(ValueError):
        s.attention(q, k, k, [3, 1])
    for scale in (0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            s.attention(q, k, k, seqs, scale=scale)
    with pytest.raises(ValueError, match="out="):
        s.attention(F((4, 4, 32), grad=True), k, k, seqs, out=q)
    for d in (4, 12, 136):
        with pytest.raises(_lib.TacoError, match="head dimension"):
            s.attention(*[F((4, 2, d))] * 3, seqs)
    with pytest.raises(_lib.TacoError, match="float64"):
        s.attention(*[F((4, 2, 32), torch.float64)] * 3, seqs)

    pages, table, lens = F((6, 16, 2, 32)), F((4, 3), torch.int32), F((4,), torch.int32)
    for args in [(q, k, None, pages, pages, table, lens), (q, F((3, 2, 32)), k, pages, pages, table, lens), (q, k, k, F((6, 16, 2, 40)), pages, table, lens),
                 (q, k, k, pages, F((5, 16, 2, 32)), table, lens), (q, k, k, pages, pages, F((4, 3), torch.int64), lens), (q, k, k, pages, pages, table, F((3,), torch.int32)),
                 (q, k, k, F((6, 16, 2, 32), torch.float16), pages, table, lens), (q, F((4, 3, 32)), F((4, 3, 32)), F((6, 16, 3, 32)), F((6, 16, 3, 32)), table, lens),
                 (q, k, k, pages, pages, F((4, 0), torch.int32), lens), (q, k, k, F((0, 16, 2, 32)), F((0, 16, 2, 32)), table, lens)]:
        with pytest.raises(ValueError):
            s.attention_step(*args)
    with pytest.raises(_lib.TacoError, match="no gradient"):
        s.attention_step(F((4, 4, 32), grad=True), k, k, pages, pages, table, lens)

    x, decay = F((4, 2, 32)), F((2,))
    with pytest.raises(ValueError):
        s.linear_attention(q, k, k, decay, seqs)
    with pytest.raises(ValueError):
        s.linear_attention(x, x, x, F((3,)), seqs)
    with pytest.raises(_lib.TacoError, match="log_decay"):
        s.linear_attention(x, x, x, F((2,), grad=True), seqs)
    with pytest.raises(ValueError):
        s.linear_attention(x, x, x, decay, seqs, state=F((1, 2, 32, 32)))
    with pytest.raises(ValueError):
        s.linear_attention(x, x, x, decay, seqs, scale=0.0)
    for state, reset in ((F((4, 2, 32, 16)), None), (F((4, 2, 32, 32), torch.float16), None), (F((4, 2, 32, 32)), F((4,), torch.float32)), (F((4, 2, 32, 32)), F((3,), torch.bool))):
        with pytest.raises(ValueError):
            s.linear_attention_step(x, x, x, decay, state, reset=reset)
    with pytest.raises(_lib.TacoError, match="no gradient"):
        s.linear_attention_step(x, x, x, decay, F((4, 2, 32, 32), grad=True))


def lists(monkeypatch, lens):
    seqs = sequence.Packed(lens, "cuda:0")
    monkeypatch.setattr(seqs, "_kept", lambda key, make: list(make()))
    return seqs


@pytest.mark.parametrize("heads", [1, 4, 200])
@pytest.mark.parametrize("lens", [[1], [0, 5, 0], [64, 65, 128, 129], [1000, 3, 33, 40000], [32] * 500, [200] * 300 + [0, 32, 33, 64] * 3])
def test_tiles_cover_every_token_once(monkeypatch, lens, heads):
    seqs = lists(monkeypatch, lens)
    seen = np.zeros(sum(lens), int)
    for rows, tiles, key_tiles, count, whole in seqs._tiles(heads):
        assert rows in (32, 128) and (rows == 32 or not whole) and (tiles[count - whole:, 1] <= 32).all() and (key_tiles[count - whole:, 1] <= 32).all() and tiles.shape == (count, 4) and tiles.dtype == np.int32
        assert sorted(map(tuple, tiles)) == sorted(map(tuple, key_tiles))
        for start, length, first, _ in tiles:
            assert first % rows == 0 and 0 <= first < length and (start, length) in set(zip(seqs.starts, seqs.lengths))
            seen[start + first:start + min(first + rows, length)] += 1
        for part in (slice(0, count - whole), slice(count - whole, count)):      # the longest first
            assert (np.diff(np.minimum(tiles[part, 2] + rows, tiles[part, 1])) <= 0).all()
            assert (np.diff(key_tiles[part, 1] - key_tiles[part, 2]) <= 0).all()
    assert (seen == 1).all()


@pytest.mark.parametrize("work", [1, 24, 5000])
@pytest.mark.parametrize("lens", [[1], [0], [256, 257, 0, 512, 513], [100000, 3], [10] * 2000 + [50000]])
def test_segments_cover_every_token_once(monkeypatch, lens, work):
    seqs = lists(monkeypatch, lens)
    table, first, count = seqs._segments(work)
    assert table.shape == (count, 8) and first[0] == 0 and first[-1] == count
    for i, n in enumerate(lens):
        mine = table[first[i]:first[i + 1]]
        assert len(mine) >= 1 and (mine[:, 0] == i).all() and (mine[:, 1] == seqs.starts[i]).all() and (mine[:, 2] == n).all()
        assert (mine[:, 3] == np.cumsum(mine[:, 4]) - mine[:, 4]).all() and mine[:, 4].sum() == n
        assert (mine[:, 4] > 0).all() or n == 0
        assert len(mine) == 1 or (mine[:-1, 4] % 64 == 0).all()


def test_page_arithmetic_on_the_host(tmp_path):
    """seq_pages.hpp, the kernel's own functions, compiled with g++ under the address sanitizer: every lookup stays inside its table and names a slot inside the cache, whatever
    the table and the lengths hold"""
    src = tmp_path / "t.cpp"
    src.write_text(r'''
#include <cassert>
#include <climits>
#include <cstdio>
#include <random>
#include <vector>
#include "seq_pages.hpp"
using namespace seq;
int main() {
    std::mt19937 r(1);
    auto pick = [&](int lo, int hi) { return (int)(lo + r() % (unsigned)(hi - lo + 1)); };
    assert(keys_of(-1, 4, 16, false) == -1 && keys_of(-1, 4, 16, true) == -1 && keys_of(INT_MIN, 4, 16, true) == -1);
    assert(keys_of(64, 4, 16, false) == 64 && keys_of(64, 4, 16, true) == -1 && keys_of(63, 4, 16, true) == 64 && keys_of(65, 4, 16, false) == -1);
    assert(keys_of(0, 1, 1, false) == 0 && keys_of(0, 1, 1, true) == 1);
    assert(keys_of(INT_MAX, INT_MAX, INT_MAX, true) == -1 && keys_of(INT_MAX, INT_MAX, INT_MAX, false) == -1);      // (room beyond 32 bits)
    assert(keys_of(1 << 30, 1 << 20, 1 << 20, true) == (1 << 30) + 1);
    assert(pieces_of(0, 256) == 1 && pieces_of(-1, 256) == 1 && pieces_of(1, 256) == 1 && pieces_of(256, 256) == 1 && pieces_of(257, 256) == 2);
    for (int n = 0; n < 20000; ++n) {
        const int width = pick(1, 6), page = pick(1, 40), pages = pick(1, 9);
        std::vector<int32_t> table(width);
        const int odd[] = {-1, INT_MIN, INT_MAX, pages, pages + 1};
        for (auto &e : table) e = pick(0, 9) < 2 ? odd[pick(0, 4)] : pick(0, pages - 1);
        const int length = pick(-3, width * page + 3);
        const bool joins = pick(0, 1);
        const int keys = keys_of(length, width, page, joins);
        assert(keys == -1 || (keys >= 0 && keys <= width * page && keys == length + (joins ? 1 : 0)));
        for (int t = 0; t < keys; ++t) {
            const Place at = place_of(table.data(), t, page, pages);
            assert(at.page >= 0 && at.page < pages && at.slot >= 0 && at.slot < page);
            assert(at.bad == (table[t / page] < 0 || table[t / page] >= pages));
            if (!at.bad) assert(at.page == table[t / page] && at.slot == t % page);
        }
    }
    assert(element_of(Place{1 << 20, 63, false}, (int64_t)1 << 14, 256) == ((int64_t)1 << 34) + 63 * 256);
    puts("ok");
}
''')
    exe = str(tmp_path / "t")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-I", os.path.join(ROOT, "taco_amd", "csrc"), "-o", exe, str(src)])
    assert subprocess.check_output([exe]).strip() == b"ok"


def test_tangents_and_scales_that_want_a_gradient_are_refused():
    """neither requires a gradient of the operands, and neither may be dropped without a word"""
    s = sequence
    x, other = torch.zeros(4, 2, 32), [torch.zeros(n) for n in ((6, 16, 2, 32), (6, 16, 2, 32))]
    table, lens, decay, state = torch.zeros(4, 3, dtype=torch.int32), torch.zeros(4, dtype=torch.int32), torch.zeros(2), torch.zeros(4, 2, 32, 32)
    seqs = s.Packed([1] * 4, "cuda:0")
    calls = [(lambda q, k, v, o: s.attention(q, k, v, seqs, out=o), [x, x, x, x]),
             (lambda q, k, v, a, b, o: s.attention_step(q, k, v, a, b, table, lens, out=o), [x, x, x] + other + [x]),
             (lambda q, k, v, g, t: s.linear_attention(q, k, v, g, seqs, state=t), [x, x, x, decay, state]),
             (lambda q, k, v, g, t, o: s.linear_attention_step(q, k, v, g, t, out=o), [x, x, x, decay, state, x])]
    with torch.autograd.forward_ad.dual_level():
        for f, args in calls:
            for i in range(len(args)):
                with pytest.raises(_lib.TacoError, match="forward-mode"):
                    f(*args[:i], torch.autograd.forward_ad.make_dual(args[i], torch.ones_like(args[i])), *args[i + 1:])
            with pytest.raises(_lib.TacoError, match="MI355X"):     # (nothing else is refused for being called here)
                f(*args)
        scale = torch.tensor(0.5)
        with pytest.raises(_lib.TacoError, match="forward-mode"):
            s._scale(torch.autograd.forward_ad.make_dual(scale, torch.ones(())), 32, True)
    q = Fake((4, 2, 32))
    for f in (lambda c: s.attention(q, q, q, seqs, scale=c), lambda c: s.linear_attention(q, q, q, Fake((2,)), seqs, scale=c)):
        with pytest.raises(_lib.TacoError, match="scale has no gradient"):
            f(torch.tensor(0.5, requires_grad=True))
    with torch.no_grad():
        assert s._scale(torch.tensor(0.5, requires_grad=True), 32, True) == 0.5


def test_sums_of_parts_only_where_tiles_of_128_rows_are():
    """a group's heads are shared out in the launch of the wide tiles alone; elsewhere no memory is asked for their sums"""
    for lens, heads, group in (([32] * 4096, 32, 8), ([64] * 4096, 16, 4), ([2000], 8, 8), ([5, 0, 31], 4, 2), ([], 4, 4), ([700, 129], 64, 32), ([700, 129], 64, 1)):
        seqs = sequence.Packed(lens, "cuda:0")
        wide = -(-np.array([n for n in lens if n > 64] + [0]) // 128).sum() * heads >= 256
        assert seqs._wide(heads) == wide and (wide or seqs._parts(heads, group, True) == seqs._parts(heads, group, False) == 1)
    assert sequence.Packed([700, 129], "cuda:0")._parts(64, 32, True) > 1


def test_whole_sequences_where_no_such_form_is(lib):
    """float32 rows above 96 have no one-launch gradients: the flag is refused, and the host layer does not set it"""
    for dim, code in ((96, 0), (104, -1), (128, -1)):
        wide = {f: tensor(ts=2 * dim, hs=dim) for f in ("q", "k", "v", "o", "d_o", "d_q", "d_k", "d_v")}
        a = attention_args(whole=1, tile_rows=32, dim=dim, n_tiles=0 if code == 0 else 1, **wide)
        assert lib.taco_attention_backward(C.byref(a), None) == code
        assert code == 0 or b"whole" in lib.taco_sequence_last_error()


@pytest.mark.parametrize("dtype,dim,flags", [(0, 96, [0, 1]), (0, 128, [0]), (1, 128, [0, 1]), (2, 128, [0, 1])])
def test_launches_of_the_gradients(monkeypatch, dtype, dim, flags):
    seqs, seen = lists(monkeypatch, [40, 5, 33, 32]), []
    monkeypatch.setattr(sequence.Packed, "_tiles", lambda self, heads, f=sequence.Packed._tiles: [(r, torch.from_numpy(t), torch.from_numpy(k), n, w) for r, t, k, n, w in f(self, heads)])
    monkeypatch.setattr(sequence, "_call", lambda f, a, device: seen.append((a.whole, a.n_tiles, a.tiles)))
    a = attention_args(dtype=dtype, dim=dim)
    sequence._launch_tiles(a, seqs, torch.device("cuda:0"), True)
    assert [x[0] for x in seen] == flags and sum(x[1] for x in seen) == 6
    assert len(seen) == 1 or seen[1][2] - seen[0][2] == 16 * seen[0][1]


def test_launches_of_fewer_than_2_to_32_threads(tmp_path):
    """seq_launches.hpp: every workgroup once, in order, and no launch whose threads pass 32 bits"""
    src = tmp_path / "t.cpp"
    src.write_text(r'''
#include <cassert>
#include <cstdio>
#include <initializer_list>
#include "seq_launches.hpp"
int main() {
    for (int threads : {64, 128, 192, 256, 384, 512})
        for (int64_t blocks : {(int64_t)0, (int64_t)1, (int64_t)8388607, (int64_t)8388608, (int64_t)16777215, (int64_t)16777216, (int64_t)16777221, (int64_t)67108864, (int64_t)2147483647}) {
            int64_t done = 0;
            int calls = 0;
            seq::in_launches(blocks, threads, [&](int32_t first, uint32_t n) {
                assert(first == done && n > 0 && (int64_t)n * threads < (int64_t)1 << 32);
                done += n;
                ++calls;
            });
            assert(done == blocks && (calls <= 1 || blocks * threads >= (int64_t)1 << 32));
        }
    puts("ok");
}
''')
    exe = str(tmp_path / "t")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-I", os.path.join(ROOT, "taco_amd", "csrc"), "-o", exe, str(src)])
    assert subprocess.check_output([exe]).strip() == b"ok"


@pytest.mark.parametrize("lens", [[2 ** 62] * 4, [2 ** 62] * 4 + [5], [2 ** 63 - 1, 1], [2 ** 31 - 4096], [2 ** 30] * 2, np.array([2 ** 63], np.uint64)])
def test_lengths_whose_sum_wraps_are_refused(lens):
    with pytest.raises(ValueError):
        sequence.Packed(lens, "cuda:0")


def test_an_output_that_requires_a_gradient_is_refused():
    """the graph that made it would go on as if nothing had been written there"""
    s, x, out = sequence, Fake((4, 2, 32)), Fake((4, 2, 32), grad=True)
    pages, table, lens = Fake((6, 16, 2, 32)), Fake((4, 3), torch.int32), Fake((4,), torch.int32)
    for f in (lambda: s.attention(x, x, x, s.Packed([4], "cuda:0"), out=out), lambda: s.attention_step(x, x, x, pages, pages, table, lens, out=out),
              lambda: s.linear_attention_step(x, x, x, Fake((2,)), Fake((4, 2, 32, 32)), out=out)):
        with pytest.raises(_lib.TacoError, match="out requires a gradient"):
            f()


def test_a_scale_whose_inverse_is_infinite_is_refused(lib):
    """the gradients of linear attention carry their states divided by it"""
    for scale, code in ((1e-40, -1), (-1e-40, -1), (2.0 ** -126, 0), (-1.0, 0)):
        for f in (lib.taco_linear_attention, lib.taco_linear_attention_backward):
            assert f(C.byref(linear_args(scale=scale, n_segments=0, n_sequences=0)), None) == code


@pytest.mark.parametrize("op", ["attention", "linear"])
@pytest.mark.parametrize("strided", [False, True])
def test_second_derivatives_are_refused(monkeypatch, op, strided):
    """a gradient that was asked for with create_graph, in a loss of its own: not a constant, also where the upstream gradient is one (a sum's).  The kernels are left out here."""
    s, seqs = sequence, sequence.Packed([3, 1], "cuda:0")
    monkeypatch.setattr(s, "_check_rows", lambda what, q, *others: (torch.device("cuda:0"), 0))
    monkeypatch.setattr(s, "_check_decay", lambda log_decay, heads, device: log_decay)
    monkeypatch.setattr(s, "_launch_tiles", lambda a, seqs, device, backward: None)
    monkeypatch.setattr(s, "_call", lambda f, a, device: None)
    monkeypatch.setattr(s.Packed, "_segments", lambda self, work: (torch.zeros(2, 8), torch.zeros(3), 2))
    leaf = [torch.randn(4, 2, 41 if strided else 32, requires_grad=True) for _ in range(3)]
    x = [t[..., :32] for t in leaf]

    def run():
        return s.attention(*x, seqs) if op == "attention" else s.linear_attention(*x, torch.zeros(2), seqs)[0]
    plain = torch.autograd.grad(run().sum(), leaf)
    for i in range(3):
        o = run()
        g, = torch.autograd.grad(o.sum(), leaf[i], create_graph=True)
        assert g.shape == plain[i].shape and g.requires_grad
        loss = o.sum() + g.square().sum()
        with pytest.raises(_lib.TacoError, match="second derivative"):
            torch.autograd.grad(loss, leaf[i], retain_graph=True)
        with pytest.raises(_lib.TacoError, match="second derivative"):
            loss.backward()
    for t in leaf:
        t.grad = None
    run().sum().backward(create_graph=True)
    for t in leaf:
        t.grad.zero_()
