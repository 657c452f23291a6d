"""Streams given to the serving calls: one of another device is refused before anything is made current."""

import pytest
import torch

from fusor_kernels import ShapeError, serving


class Stream:
    def __init__(self, index):
        self.device = torch.device("cuda", index)


def test_a_stream_of_another_device_is_refused():
    serving._load()
    with pytest.raises(ShapeError, match="a stream of cuda:1, the tensors are on cuda:0"):
        serving._place(torch.device("cuda", 0), Stream(1))
    with pytest.raises(ShapeError, match="a stream of cuda:0"):
        serving._place(torch.device("cuda", 1), Stream(0))
    serving._place(torch.device("cuda", 1), Stream(1))  # (a context that is not entered)
