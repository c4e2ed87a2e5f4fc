"""The work lists of the shared-prefix attention, on the CPU.

csrc/prefix_plan.h is plain C++: tests/c/prefix_plan_check.cpp is compiled with
it and goes through every (row, key) pair of a shape: each kept pair is in one
tile, every dropped one in a masked tile, every dropped one that the tensor
holds in a guarded tile, and nothing is kept where a tile has no scores."""
import os
import random
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "qwen3-embedding-webgpu-prepacked_b200", "csrc")


@pytest.fixture(scope="module")
def plan_check(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("plan") / "prefix_plan_check")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-I", CSRC,
                    os.path.join(HERE, "c", "prefix_plan_check.cpp"), "-o", exe], check=True)
    return exe


def check(exe, prefix, sparse, sparse_prefix, window, group, requests):
    """[kept pairs, tiles] of blocks of two row tiles; blocks of one are checked too."""
    for row_tiles in (1, 2):
        args = [prefix, sparse, sparse_prefix, window, group, row_tiles]
        for n, m in requests:
            args += [n, m]
        out = subprocess.run([exe] + [str(a) for a in args], capture_output=True, text=True)
        assert out.returncode == 0, (args, out.stdout)
    return [int(x) for x in out.stdout.split()]


@pytest.mark.parametrize("prefix", [0, 1, 16, 128, 176, 500])
@pytest.mark.parametrize("sparse", [0, 1])
@pytest.mark.parametrize("group", [1, 2, 3, 8, 128])
def test_ragged_batch(plan_check, prefix, sparse, group):
    check(plan_check, prefix, sparse, 176, 432, group, [(17, 17), (1, 1), (0, 0), (150, 150), (3, 90),
                                                     (0, 40), (64, 300)])


def test_random_shapes(plan_check):
    r = random.Random(5)
    for _ in range(150):
        requests = []
        for _ in range(r.randrange(1, 9)):
            n = r.choice([0, 1, 2, r.randrange(1, 200)])
            requests.append((n, n + r.choice([0, 0, 1, r.randrange(0, 200)])))
        check(plan_check, r.choice([0, 1, r.randrange(1, 700)]), r.randrange(2),
              r.choice([0, 1, 16, 170, 176, 900]), r.choice([1, 2, 100, 432]),
              r.choice([1, 2, 3, 4, 5, 8, 16, 100]), requests)


def test_work_of_the_binding(pkg, plan_check):
    cu_q, cu_k = [0, 100, 101, 161], [0, 100, 151, 511]
    requests = [(100, 100), (1, 51), (60, 360)]
    for mode, sparse in ((pkg.attention.MODE_FULL, 0), (pkg.attention.MODE_SPARSE, 1)):
        pairs, tiles = pkg.prefix.prefix_attention_work(cu_q, 300, 16, 8, cu_k, mode)
        assert [pairs, tiles // 8] == check(plan_check, 300, sparse, 176, 432, 2, requests)


def test_work_without_prefix_is_causal_attention(pkg):
    cu = [0, 5000, 5500, 5501, 7000]
    for mode in (pkg.attention.MODE_AUTO, pkg.attention.MODE_FULL, pkg.attention.MODE_SPARSE):
        assert pkg.prefix.prefix_attention_work(cu, 0, 16, 8, mode=mode)[0] == \
            pkg.attention.attention_work(cu, mode)[0]


@pytest.mark.parametrize("bad", [
    dict(cu_seqlens=[0, 5], cu_seqlens_k=[0, 4]),          # more queries than keys
    dict(cu_seqlens=[0, 5, 3]),                            # decreasing
    dict(cu_seqlens=[1, 5]),                               # does not begin at 0
    dict(cu_seqlens=[0, 5], prefix_len=-1),
    dict(cu_seqlens=[0, 5], prefix_len=1 << 30),           # positions past 2^30
    dict(cu_seqlens=[0, 5], q_heads=12),                   # not a multiple of kv_heads
    dict(cu_seqlens=[0, 5], q_heads=129, kv_heads=1),
    dict(cu_seqlens=[0, 5], q_heads=4),                    # fewer than kv_heads
    dict(cu_seqlens=[0, 5], mode=3),
    dict(cu_seqlens=[0, 5], window=0),
    dict(cu_seqlens=[0, 5], sparse_prefix=-1),
])
def test_refusals(pkg, bad):
    args = dict(dict(cu_seqlens=[0, 5], prefix_len=10, q_heads=16, kv_heads=8), **bad)
    with pytest.raises(pkg._lib.QwaError):
        pkg.prefix.prefix_attention_work(**args)


def test_requests_of_q_and_k_must_agree(pkg):
    with pytest.raises(ValueError):
        pkg.prefix.prefix_attention_work([0, 5], 10, 16, 8, [0, 5, 6])


@pytest.mark.parametrize("bad", [dict(prefix_len=2 ** 32), dict(window=2 ** 32 + 5),
                                 dict(sparse_prefix=-2 ** 32), dict(q_heads=2 ** 32 + 16),
                                 dict(cu_seqlens=[0, 2 ** 32 + 5])])
def test_numbers_past_32_bits_are_refused(pkg, bad):
    args = dict(cu_seqlens=[0, 5], prefix_len=10, q_heads=16, kv_heads=8)
    args.update(bad)
    with pytest.raises(ValueError):
        pkg.prefix.prefix_attention_work(**args)


def test_offsets_of_a_tensor_count_by_value(pkg):
    import torch
    cu = torch.tensor([0, 5, 40], dtype=torch.int32)
    assert pkg.prefix._lengths(cu) == (0, 5, 40)
    assert pkg.prefix.prefix_attention_work(cu, 10, 16, 8) == \
        pkg.prefix.prefix_attention_work([0, 5, 40], 10, 16, 8)
