"""Every kernel that takes an 8-bit product, each against a reference in 64 bits.

Which kernel takes a product follows from estimated times, so a list of sizes says little about what it runs.  Each case here
names the kernel it is for (as ``tca_int8_linear_way`` numbers them: 0 to 13 tiles for aligned rows, 16 to 22 for rows at any
address, 32 more where the operands are copied first).  That it still goes there is asserted without a GPU; the products run
on one."""
import threading

import pytest
import torch

from triton_client_amd import _native
from triton_client_amd.ops import int8

from test_gpu_int8 import TYPES, _linear_reference

# Tiles of a large product (0: 256 x 256, 1: 256 x 128, 2: 128 x 128, 3: 64 x 128, 4: 64 x 64): rows of outputs of whole
# lines (n a multiple of 64), of whole 16-byte pieces (of 8), and at any address; an odd and an even number of stages of 128 k;
# more tiles than the card holds at a time.  The last rows and columns of tiles are never full.
TILES = [
    (0, 3978, 3231, 656), (0, 2490, 4979, 784), (0, 6449, 4655, 672), (0, 4354, 2752, 144), (0, 1943, 6208, 272),
    (0, 5652, 5056, 144), (0, 5609, 2184, 144), (0, 6168, 1944, 272), (0, 4777, 6152, 144),
    (1, 2568, 1540, 2032), (1, 654, 6138, 2096), (1, 6550, 2374, 1936), (1, 641, 6080, 912), (1, 788, 5056, 1040),
    (1, 2324, 6464, 1008), (1, 1649, 2520, 912), (1, 2371, 1704, 1072), (1, 5513, 2824, 960),
    (2, 1041, 4826, 144), (2, 709, 6868, 16), (2, 1289, 6983, 16), (2, 3401, 1216, 144), (2, 577, 6656, 16), (2, 6539, 1216, 16),
    (2, 706, 5456, 144), (2, 580, 6560, 16), (2, 6574, 1160, 16),
    (3, 1034, 2893, 144), (3, 6983, 387, 16), (3, 1292, 5925, 16), (3, 515, 5568, 144), (3, 449, 6208, 16), (3, 1160, 6592, 16),
    (3, 461, 6200, 144), (3, 6978, 392, 16), (3, 5391, 1416, 16),
    (4, 4119, 68, 144), (4, 6146, 33, 16), (4, 579, 6542, 16), (4, 211, 1792, 144), (4, 49, 6208, 16), (4, 4125, 72, 144),
    (4, 4101, 72, 16),
]

# k shared by the waves of a block, through rings filled by DMA
SPLIT = [
    (5, 81, 2789, 528), (5, 307, 832, 928), (5, 1748, 208, 528), (6, 4167, 18, 816), (6, 145, 832, 1424), (6, 2084, 88, 784),
    (7, 692, 81, 784), (7, 194, 320, 912), (7, 33, 1368, 816), (8, 417, 297, 784), (8, 338, 384, 912), (8, 311, 416, 784),
    (9, 8, 4121, 1616), (9, 1, 4160, 944), (9, 1, 4128, 784), (10, 404, 468, 272), (10, 225, 832, 144), (10, 559, 344, 272),
    (11, 5, 272, 3024), (11, 1, 1, 1696), (11, 1, 64, 1552), (12, 317, 3, 1088), (12, 1, 64, 400), (12, 1, 8, 272),
    (13, 23, 228, 16), (13, 81, 704, 272), (13, 1, 8, 144),
    # weights past the caches; weight rows multiples of 8 KB apart
    (12, 7, 33000, 4096), (12, 16, 16400, 8192),
]

# rows at any address, as they are
ANY = [
    (16, 219, 4397, 2306), (16, 135, 5632, 1415), (16, 130, 6176, 1799), (17, 194, 639, 1720 + 1), (17, 49, 3136, 641),
    (17, 273, 688, 516), (18, 4125, 70, 390), (18, 179, 1408, 392), (18, 559, 472, 264), (19, 438, 593, 257), (19, 34, 4224, 711),
    (19, 33, 4336, 538), (20, 17, 43, 2846), (20, 1, 64, 513), (20, 1, 8, 641), (21, 31, 588, 4), (21, 1, 64, 129), (21, 1, 1, 1),
    (22, 933, 278, 130), (22, 33, 5760, 1), (22, 263, 992, 130),
]

# copied to aligned rows first
COPIED = [
    (32, 4597, 2701, 642), (32, 3402, 3648, 129), (32, 2061, 5784, 275), (33, 2381, 1686, 1966), (33, 779, 5312, 907),
    (33, 1559, 2584, 1029), (34, 5169, 1171, 1), (34, 783, 6336, 132), (34, 4050, 1296, 129), (35, 3727, 839, 517),
    (35, 1665, 4672, 129), (35, 1544, 5000, 1), (36, 299, 1694, 1926), (36, 625, 832, 1834), (36, 801, 656, 1797),
    (37, 835, 292, 2811), (37, 697, 384, 2674), (38, 204, 636, 4281), (39, 187, 1347, 2755), (39, 828, 304, 2148),
    (40, 199, 2368, 1987), (40, 261, 1912, 2860), (45, 839, 296, 4156),
]

CASES = TILES + SPLIT + ANY + COPIED


def _way(m, n, k, x=0, w=0, pad=0):
    """The kernel of a product of contiguous operands; outputs, and a residual, ``pad`` further apart than their rows."""
    return _native.hip().tca_int8_linear_way(x, w, m, n, k, k, k, n + pad if pad else 0, n + pad)


def _workspace(m, n, k):
    return _native.hip().tca_int8_linear_workspace_bytes(0, 0, m, n, k, k, k)


def test_the_cases_reach_the_kernels_that_they_name():
    for way, m, n, k in CASES:
        assert _way(m, n, k) == _way(m, n, k, pad=64) == way, (m, n, k)
        assert (_workspace(m, n, k) > 0) == (way >= 32), (m, n, k)


def test_every_kernel_has_cases():
    ways = {way % 32 for way, *_ in CASES}
    assert ways == {*range(14), *range(16, 23)}
    resident = {0: (256, 256, 256), 1: (256, 128, 256), 2: (128, 128, 512), 3: (64, 128, 512), 4: (64, 64, 1024)}
    for way, (rows, columns, most) in resident.items():
        mine = [case[1:] for case in TILES if case[0] == way]
        assert {((n % 64 == 0) + (n % 8 == 0), (k + 127) // 128 % 2) for _, n, k in mine} == {(r, s) for r in range(3) for s in range(2)}
        assert any(-(-m // rows) * -(-n // columns) > most for m, n, _ in mine)
    for m, n, k in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (1, 1, int8.MAX_K + 1)):
        assert _way(m, n, k) == -1


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _operands(m, n, k, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x, w = (torch.randint(-128, 128, shape, generator=g, dtype=torch.int8, device="cuda") for shape in ((m, k), (n, k)))
    xs, ws = _normal(g, m).abs() * 0.01 + 1e-3, _normal(g, n).abs() * 1e-3 + 1e-4
    return x, xs, w, ws, _normal(g, n).to(dtype), _normal(g, m, n).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("way,m,n,k", CASES)
def test_each_kernel(way, m, n, k, dtype):
    """Without and with bias and residual; what lies around the outputs stays."""
    x, xs, w, ws, b, r = _operands(m, n, k, dtype)
    for bias, residual, pad in ((None, None, 0), (b, r, 0), (None, r, 64), (b, None, 64)):
        rows = torch.full((m + 2, n + pad), 7.0, dtype=dtype, device="cuda")
        out = rows[1:-1, :n]
        if residual is not None and pad:
            wide = torch.zeros(m, n + pad, dtype=dtype, device="cuda")
            wide[:, :n] = residual
            residual = wide[:, :n]
        assert _way(m, n, k, x.data_ptr(), w.data_ptr(), pad) == way
        int8.linear_int8(x, xs, w, ws, bias=bias, residual=residual, out=out)
        ref, slack = _linear_reference(x, xs, w, ws, bias, residual, dtype)
        assert ((out.double() - ref).abs() <= slack).all()
        assert (rows[0] == 7).all() and (rows[-1] == 7).all() and (rows[:, n:] == 7).all()
        plain = int8.linear_int8(x, xs, w, ws, bias=bias, residual=residual, dtype=dtype)
        assert torch.equal(plain, out)


# sizes whose operands are copied to a workspace of the call
WITH_WORKSPACE = [(1100, 1201, 1333), (2500, 2600, 399)]


def test_the_workspace_cases_have_one():
    for size in WITH_WORKSPACE:
        assert _workspace(*size) > 0, size


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", WITH_WORKSPACE)
def test_workspaces_of_two_threads(m, n, k):
    """Calls of two threads, each on a stream of its own, their workspaces in flight at the same time."""
    cases = []
    for seed in range(2):
        x, xs, w, ws, _, _ = _operands(m, n, k, torch.bfloat16, seed)
        want = int8.linear_int8(x, xs, w, ws, dtype=torch.bfloat16)
        ref, slack = _linear_reference(x, xs, w, ws, None, None, torch.bfloat16)
        assert ((want.double() - ref).abs() <= slack).all()
        cases.append((x, xs, w, ws, want))
    torch.cuda.synchronize()
    bad = []

    def work(x, xs, w, ws, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    if not torch.equal(int8.linear_int8(x, xs, w, ws, dtype=torch.bfloat16), want):
                        bad.append("a result differs")
        except Exception as e:  # noqa: BLE001 - reported by the test's own thread
            bad.append(repr(e))

    threads = [threading.Thread(target=work, args=c) for c in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", WITH_WORKSPACE)
def test_workspaces_in_graphs(m, n, k):
    """Captured twice; replayed with eager calls between, and on two streams at the same time."""
    x, xs, w, ws, _, _ = _operands(m, n, k, torch.float16)
    inputs = [torch.roll(x, shift, 0) for shift in range(3)]
    want = [int8.linear_int8(t, xs, w, ws) for t in inputs]
    ref, slack = _linear_reference(inputs[1], xs, w, ws, None, None, torch.float16)
    assert ((want[1].double() - ref).abs() <= slack).all()
    graphs = []
    for _ in range(2):
        x_in = inputs[0].clone()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = int8.linear_int8(x_in, xs, w, ws)
        graphs.append((graph, x_in, y))
    for turn in range(6):
        for i, (graph, x_in, y) in enumerate(graphs):
            at = (turn + i) % 3
            x_in.copy_(inputs[at])
            graph.replay()
            assert torch.equal(int8.linear_int8(inputs[at], xs, w, ws), want[at])
            assert torch.equal(y, want[at])
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(3):
        for i, (_, x_in, _) in enumerate(graphs):
            x_in.copy_(inputs[(turn + i) % 3])
        torch.cuda.synchronize()
        for stream, (graph, _, _) in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for i, (_, _, y) in enumerate(graphs):
            assert torch.equal(y, want[(turn + i) % 3])
