"""What a PackedSequences object does not let happen to it: the kernels have its arrays' addresses from the start, so another
array put in an attribute's place would be ignored, and the old one's memory be read after it was freed."""
import pytest
import torch

NAMES = ["cu_q", "cu_k", "len_k", "pos_q", "pos_k", "batch", "causal", "buckets", "device", "_lut", "_c", "_ref"]


@pytest.fixture
def seqs(monkeypatch):
    from imageni2r_amd import packed
    monkeypatch.setattr(packed, "_index", lambda t, *a: t)  # (no kernel runs: the arrays may lie on the host)
    cu = torch.tensor([0, 4, 9], dtype=torch.int32)
    return packed.PackedSequences(cu, cu.clone(), len_k=torch.tensor([1, 2], dtype=torch.int32))


@pytest.mark.parametrize("name", NAMES)
def test_attributes_are_fixed(seqs, name):
    held = getattr(seqs, name)
    with pytest.raises(AttributeError, match=f"PackedSequences.{name} is fixed"):
        setattr(seqs, name, held.clone() if isinstance(held, torch.Tensor) else object())
    with pytest.raises(AttributeError, match=f"PackedSequences.{name} is fixed"):
        delattr(seqs, name)
    assert getattr(seqs, name) is held


def test_values_are_not(seqs):
    at = seqs.len_k.data_ptr()
    seqs.len_k.copy_(torch.tensor([3, 4], dtype=torch.int32))
    seqs.len_k += 1
    assert seqs.len_k.tolist() == [4, 5] and seqs._c.len_k == at


def test_names_of_the_class():
    from imageni2r_amd import packed
    assert [f[0] for f in packed._Seqs._fields_[:5]] == NAMES[:5]
