"""Sizes at which the cache and attention entry points' 32-bit quantities end: refused before a launch. Addresses are made up:
nothing is launched, so nothing reads them."""
from heterofusedkernels_amd import capi
from test_cache_boundary_cpu import attention, plane, rows

TOO_LARGE = -3


def both_workspaces(a):
    return capi.prompt_attention_workspace(a, 1, 2)[0], capi.prefix_attention_workspace(a, 2, 2)[0]


def test_blocks_whose_span_wraps_in_64_bits():
    """Token strides whose products with a block's last token are 2^64 and a little, or many times that."""
    for stride, T in ((1 << 35, (1 << 28) + 1), (1 << 37, (1 << 26) + 1), ((1 << 35) + 8, (1 << 28) + 1), (1 << 39, 1 << 28), ((1 << 40) - 8, 1 << 29)):
        assert both_workspaces(attention(k=plane(T=T, blocks=1, strides=(0, stride, 64)))) == (TOO_LARGE, TOO_LARGE)
        a = attention(k=plane(T=T, blocks=1, kind=capi.FP8_E4M3, scales=4096, strides=(0, 128, 64)))
        for side in (a.k, a.v):
            side.scale_token_stride = stride
        assert both_workspaces(a) == (TOO_LARGE, TOO_LARGE)
    # the longest block there is, one token further, and a block of one token, whose stride means nothing
    most = (0xffffffff // 2) & ~7
    assert both_workspaces(attention(k=plane(T=2, blocks=1, strides=(0, most, 64)))) == (0, 0)
    assert both_workspaces(attention(k=plane(T=2, blocks=1, strides=(0, most + 8, 64)))) == (TOO_LARGE, TOO_LARGE)
    assert both_workspaces(attention(k=plane(T=1, blocks=1, strides=(0, 1 << 39, 64)))) == (0, 0)


def test_launches_of_2_to_the_32_threads():
    """The runtime takes no launch of as many threads. 16 lanes have a row of 128 values in 16 bits, 8 in e4m3, 64 have one of 512
    that is taken value by value; 512 threads have 256 query rows of a prompt, 64 a joined row."""
    for call in (capi.cache_write, capi.cache_read):
        assert call(plane(dim=128), rows(dim=128), None, None, 8, 1 << 27) == TOO_LARGE
        assert call(plane(dim=128), rows(dim=128), plane(dim=128), rows(dim=128), 8, 1 << 26) == TOO_LARGE      # both sides together
        assert call(plane(dim=128, kind=capi.FP8_E4M3, scales=64), rows(dim=128), None, None, 8, 1 << 28) == TOO_LARGE
        assert call(plane(dim=512), rows(data=4098, dim=512), None, None, 8, 1 << 25) == TOO_LARGE
    space, size = 256, 1 << 62
    a = attention(n=1 << 23)      # every sequence's last tile of rows counts
    assert capi.prompt_attention(a, 8, 1 << 23, 1, 8, 8, True, space, size) == TOO_LARGE
    a = attention(n=1 << 24)
    assert capi.prefix_attention(a, 8, 1, 8, 8, 1, 8, space, size) == TOO_LARGE
    assert capi.prefix_attention(a, 0, 0, 0, 8, 1, 8, space, size) == TOO_LARGE
