"""The cases of test_gpu_tree and test_gpu_tree_shapes with the tensor-core kernels asked for by name, so that none is answered on the
CUDA cores unnoticed."""
import pytest
import torch

import test_gpu_tree as cases
import test_gpu_tree_shapes as shapes

pytestmark = pytest.mark.gpu
KERNELS = torch.bfloat16, 'sm100'


@pytest.mark.parametrize('b, t, hq, hkv, d', [(1, 1, 1, 1, 64), (2, 1, 32, 4, 64), (3, 7, 8, 2, 64), (2, 16, 16, 4, 128), (1, 33, 12, 4, 32), (2, 5, 8, 8, 80),
                                              (1, 64, 8, 1, 128), (2, 9, 14, 2, 96), (1, 130, 4, 2, 64), (1, 3, 5, 1, 8)])
def test_shapes(b, t, hq, hkv, d):
    cases.test_shapes(*KERNELS, b, t, hq, hkv, d)


@pytest.mark.parametrize('length', [0, 1, 63, 64, 65, 127, 128, 129, 257, 500])
def test_lengths_around_the_blocks(length):
    cases.test_lengths_around_the_blocks(*KERNELS, length)


@pytest.mark.parametrize('b', [1, 5, 37, 70])
def test_ragged_batches(b):
    cases.test_ragged_batches(*KERNELS, b)


def test_masks_that_leave_rows_empty():
    cases.test_masks_that_leave_rows_empty(*KERNELS)


@pytest.mark.parametrize('garbage', [float('nan'), float('inf'), -float('inf'), 3e38])
def test_what_nobody_sees_leaves_no_trace(garbage):
    cases.test_what_nobody_sees_leaves_no_trace(*KERNELS, garbage)


def test_large_logits():
    cases.test_large_logits(*KERNELS)


@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('t, g', [(1, 8), (2, 4), (1, 9), (1, 16), (16, 1), (1, 17), (4, 8), (11, 3), (1, 40), (16, 4), (13, 5), (32, 4), (43, 3), (64, 4), (65, 4), (97, 4)])
def test_rows_around_the_tiles(d, t, g):
    shapes.test_rows_around_the_tiles(*KERNELS, d, t, g)


@pytest.mark.parametrize('t, hq, hkv', [(300, 4, 1), (513, 2, 2)])
def test_long_chains(t, hq, hkv):
    shapes.test_long_chains(*KERNELS, t, hq, hkv)


def test_drafts_of_a_padded_batch():
    shapes.test_drafts_of_a_padded_batch(*KERNELS)
