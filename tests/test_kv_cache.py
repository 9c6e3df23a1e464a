"""Host side of the quantised key / value cache: sizes and refusals that need no GPU."""
import pytest


@pytest.mark.parametrize("qtype", [2, 3, 8])
@pytest.mark.parametrize("heads,d,page,pages", [(1, 64, 16, 1), (5, 128, 48, 7), (8, 256, 5184, 3)])
def test_bytes_are_those_of_the_formats_rows(s3b, qtype, heads, d, page, pages):
    assert s3b.kv_cache_bytes(qtype, heads, d, page, pages) == 2 * s3b.row_size(qtype, d) * heads * page * pages


@pytest.mark.parametrize("qtype,heads,d,page,pages", [
    (1, 1, 64, 16, 1), (2, 0, 64, 16, 1), (2, -1, 64, 16, 1), (2, 1, 96, 16, 1), (2, 1, 32, 16, 1), (2, 1, 64, 0, 1),
    (2, 1, 64, 24, 1), (2, 1, 64, -16, 1), (2, 1, 64, 16, 0), (2, 1, 64, 16, -1), (8, 2 ** 30, 256, 2 ** 30, 1),
    (2, 2 ** 20, 64, 2 ** 20, 2 ** 62)])
def test_bytes_refuses(s3b, qtype, heads, d, page, pages):
    with pytest.raises(s3b.S3BError):
        s3b.kv_cache_bytes(qtype, heads, d, page, pages)
