"""What the decoder's layers refuse before anything is put on a device."""
import numpy as np
import pytest

from adhip.decoder import DecoderAttention, DecoderRecurrence

X = np.zeros((2, 5, 8), np.float32)


def layers(documents):
    yield lambda: DecoderAttention(None, X, X, 2, 1, 8, documents=documents)
    yield lambda: DecoderRecurrence(None, X, X, 16, documents=documents)


@pytest.mark.parametrize("documents", [np.full((2, 5), 1 << 32), np.full((2, 5), -(1 << 40)), [[0.5] * 5] * 2])
def test_numbers_of_documents_keep_their_value(documents):
    """Cut off to 32 bits, hashes of 64 would meet others: one document to the masks."""
    for layer in layers(documents):
        with pytest.raises(ValueError, match="32 bits"):
            layer()


def test_documents_of_another_shape():
    for layer in layers(np.zeros((2, 6), np.int32)):
        with pytest.raises(ValueError, match="shape"):
            layer()
