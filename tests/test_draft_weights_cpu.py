"""The oracle of verification where probabilities are negative or no numbers."""
import torch

from oracle import drafts as od


def test_they_count_as_zeros_of_either_side():
    nan = float("nan")
    p = torch.tensor([[[0.25, 0.25, 0.25, 0.25, -1.0], [0.0, nan, 0.5, -2.0, 0.0]]])
    q = torch.tensor([[[0.5, -8.0, nan, 0.25, -4.0]]])
    for u, want in ((0.0, 1), (0.49, 1), (0.5, 2), (0.9999, 2)):         # left of the target: 0, 0.25, 0.25, 0, 0
        assert od.verify(p, torch.tensor([[0]]), torch.tensor([[0.75, u]]), q) == ([0], [[want, -1]])
    for x, k in ((4, 0), (2, 1), (1, 1), (3, 1)):
        tokens = [[1, -1]] if k == 0 else [[x, 2]]
        assert od.verify(p, torch.tensor([[x]]), torch.tensor([[0.75, 0.0]]), q) == ([k], tokens)
