"""More rows than the C struct's 32 bits hold are refused, not taken modulo 2^32 (without a GPU)."""

from types import SimpleNamespace

import pytest
import torch

from opac1ty_b200 import int8

MOST = 2**31 - 4096


class Codes:
    """What Int8Rows asks of a tensor of codes [rows, 16]."""
    dtype, device, is_cuda = torch.int8, torch.device("cuda", 0), True

    def __init__(self, rows):
        self.shape = (rows, 16)

    def dim(self):
        return 2

    def stride(self, i=None):
        return (16, 1) if i is None else (16, 1)[i]

    def data_ptr(self):
        return 4096

    def get_device(self):
        return 0


def scales(rows):
    return SimpleNamespace(dtype=torch.float32, shape=(rows,), device=Codes.device, stride=lambda i: 1, data_ptr=lambda: 4096)


@pytest.mark.parametrize("rows", [MOST + 1, 2**31, 2**32 - 1, 2**32, 2**32 + 5])
def test_more_rows_than_the_struct_holds(rows):
    with pytest.raises(ValueError, match="rows"):
        int8.Int8Rows(Codes(rows), scales(rows))
    for n in (1, 4096):
        with pytest.raises(ValueError, match="rows"):
            int8.Int8Rows._new(None, rows, n, None)


def test_the_most():
    r = int8.Int8Rows(Codes(MOST), scales(MOST))
    assert r.c.rows == r.rows == MOST
