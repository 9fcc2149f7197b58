"""Shapes that take the forms of the search operators which small batches do not,
with the form that each is meant to take: a rule that moves fails a test, on the
host and on the GPU."""
import ctypes as C

from ane import _lib

lib = _lib.load()
AT = 0x10000  # an address that is never followed


def _form(n, call, *args):
    out = (C.c_int32 * n)()
    rc = call(*args, out)
    assert rc == _lib.ANE_OK, lib.ane_op_last_error().decode()
    return tuple(out)


def _cache(kvh, dh, P, pages=500):
    return _lib.Kv8Cache(AT, AT, AT, AT, pages, P, kvh, dh, 0)


def _batch(lens, width, rows_behind, max_len=0, max_new=0):
    return _lib.Kv8Batch(AT, AT, AT, width, width, len(lens), sum(n for _, n in lens) + rows_behind, max_len, max_new)


def width_of(lens, P, spare):
    return max(-(-(held + new) // P) for held, new in lens) + spare


def select_form(lens, heads, kvh, dh, P, spare=1, rows_behind=2, **hints):
    """(tiles of 16 query rows, tokens a block, waves, in parts, scores in LDS)"""
    return _form(5, lib.ane_debug_kv8_select_form, _cache(kvh, dh, P),
                 _batch(lens, width_of(lens, P, spare), rows_behind, **hints), heads)


# The choice of pages: {lens: (held, new) of each sequence, ...}, the form, and how the scores of the longest context
# are held: in registers, in LDS, or made again in every pass (where the hint is of a shorter one).
def _chunk(pages, P=16):
    return [(P * pages - 90, 89), (70, 69), (P * pages - 300, 143)]


def _tokens(n, pages, P=16):
    return [(P * pages - 1 - 7 * i if i < 40 else P * (i * 37 % pages) + i % P, 1) for i in range(n)]


SELECT = [
    # chunks, four tokens a block: groups of 1 to 4
    (dict(lens=_chunk(70), heads=6, kvh=2, dh=64, P=16), (1, 4, 4, 0), "registers"),
    (dict(lens=_chunk(70), heads=8, kvh=2, dh=128, P=16), (1, 4, 4, 0), "registers"),
    (dict(lens=_chunk(1100), heads=6, kvh=2, dh=64, P=16), (1, 4, 4, 0), "LDS"),
    (dict(lens=_chunk(1100), heads=2, kvh=2, dh=128, P=16), (1, 4, 4, 0), "LDS"),
    (dict(lens=_chunk(1100), heads=8, kvh=2, dh=64, P=16, max_len=100), (1, 4, 4, 0), "again"),
    (dict(lens=_chunk(300), heads=6, kvh=2, dh=128, P=16, max_len=100, max_new=143), (1, 4, 4, 0), "again"),
    # two tokens a block: groups of 5 to 8, more than 64 pages
    (dict(lens=_chunk(70), heads=12, kvh=2, dh=64, P=16), (1, 2, 4, 0), "registers"),
    (dict(lens=_chunk(70), heads=16, kvh=2, dh=128, P=16), (1, 2, 4, 0), "registers"),
    (dict(lens=_chunk(1100), heads=16, kvh=2, dh=64, P=16), (1, 2, 4, 0), "LDS"),
    (dict(lens=_chunk(1100), heads=10, kvh=2, dh=128, P=16), (1, 2, 4, 0), "LDS"),
    (dict(lens=_chunk(1100), heads=10, kvh=2, dh=64, P=16, max_len=16 * 66), (1, 2, 4, 0), "again"),
    (dict(lens=_chunk(300), heads=12, kvh=2, dh=128, P=16, max_len=16 * 66, max_new=143), (1, 2, 4, 0), "again"),
    # a wave a token: up to 64, 256 and 512 pages by the number of lists
    (dict(lens=_tokens(150, 250), heads=8, kvh=4, dh=64, P=16, max_new=1), (1, 1, 1, 0), "registers"),
    (dict(lens=_tokens(150, 250), heads=8, kvh=4, dh=128, P=16, max_new=1), (1, 1, 1, 0), "registers"),
    (dict(lens=_tokens(300, 500), heads=12, kvh=4, dh=64, P=16, max_new=1), (1, 1, 1, 0), "registers"),
    (dict(lens=_tokens(150, 500), heads=160, kvh=8, dh=128, P=16, max_new=1), (2, 1, 1, 0), "registers"),
    (dict(lens=_tokens(300, 500), heads=4, kvh=4, dh=64, P=16, max_len=16 * 100, max_new=1), (1, 1, 1, 0), "again"),
    (dict(lens=_tokens(300, 1300), heads=4, kvh=4, dh=64, P=16, max_len=16 * 500, max_new=1), (1, 1, 1, 0), "again"),
    # four waves
    (dict(lens=_tokens(40, 300), heads=4, kvh=2, dh=128, P=16, max_new=1), (1, 1, 4, 0), "registers"),
    (dict(lens=_tokens(40, 300), heads=40, kvh=2, dh=64, P=16, max_new=1), (2, 1, 4, 0), "registers"),
    (dict(lens=_tokens(40, 300), heads=34, kvh=2, dh=128, P=16, max_new=1), (2, 1, 4, 0), "registers"),
    (dict(lens=_tokens(40, 1200), heads=4, kvh=2, dh=64, P=16, max_len=16 * 100, max_new=1), (1, 1, 4, 0), "again"),
    (dict(lens=_tokens(40, 700), heads=34, kvh=2, dh=128, P=16, max_len=16 * 100, max_new=1), (2, 1, 4, 0), "again"),
    # eight waves
    (dict(lens=_tokens(150, 900), heads=6, kvh=2, dh=128, P=16, max_new=1), (1, 1, 8, 0), "registers"),
    (dict(lens=_tokens(150, 900), heads=40, kvh=2, dh=64, P=16, max_new=1), (2, 1, 8, 0), "registers"),
    (dict(lens=_tokens(150, 900), heads=64, kvh=2, dh=128, P=16, max_new=1), (2, 1, 8, 0), "registers"),
    (dict(lens=_tokens(150, 1500), heads=2, kvh=2, dh=128, P=16, max_new=1), (1, 1, 8, 0), "LDS"),
    (dict(lens=_tokens(150, 1500), heads=34, kvh=2, dh=64, P=16, max_new=1), (2, 1, 8, 0), "LDS"),
    (dict(lens=_tokens(40, 1500), heads=2, kvh=2, dh=64, P=16, max_len=16 * 600, max_new=1), (1, 1, 8, 0), "again"),
    (dict(lens=_tokens(150, 1500), heads=34, kvh=2, dh=128, P=16, max_len=16 * 600, max_new=1), (2, 1, 8, 0), "again"),
]
HELD = 1024  # pages whose scores registers hold


def where_scores_are(shape, form):
    """Of the tile with the longest context."""
    held, new = max(shape["lens"], key=sum)
    pages = -(-(held + new) // shape["P"])
    if min(form[1], new) * (-(-pages // 64) * 64) > form[4]:
        return "again"
    return "registers" if pages <= HELD else "LDS"


def name_of(case):
    shape, form, *rest = case
    return "-".join([f"{shape['heads']}-{shape['kvh']}-{shape['dh']}", *(str(x) for x in form), *(str(x) for x in rest)])


def attend_form(lens, heads, kvh, dh, P, count, spare=1, rows_behind=2, **hints):
    """(tiles of 16 rows, tokens a tile, waves on its keys, parts, longest first, places with masks)"""
    return _form(6, lib.ane_debug_kv8_attend_form, _cache(kvh, dh, P),
                 _batch(lens, width_of(lens, P, spare), rows_behind, **hints), heads, count)


# Attention over lists of `count` pages: the form as (tiles of 16 rows, whether tokens share a tile, waves, whether
# its keys are cut, longest contexts first).
ATTEND = [
    # a wave a list, pages of at least a step's 32 keys and smaller ones
    (dict(lens=[(700, 1)] * 201, heads=12, kvh=4, dh=64, P=32, count=7, max_new=1), (1, False, 1, False, 0)),
    (dict(lens=[(400, 1)] * 101, heads=16, kvh=8, dh=128, P=16, count=10, max_new=1), (1, False, 1, False, 0)),
    (dict(lens=[(500, 781)], heads=24, kvh=1, dh=128, P=64, count=5), (2, False, 1, False, 0)),
    (dict(lens=[(900, 60), (3, 170), (0, 191)], heads=40, kvh=2, dh=64, P=16, count=13), (2, False, 1, False, 0)),
    # lists that are cut, pages smaller than a step
    (dict(lens=[(16 * 100, 1), (40, 2)], heads=16, kvh=2, dh=128, P=16, count=80), (1, False, 4, True, 0)),
    (dict(lens=[(16 * 140, 1), (40, 2)], heads=40, kvh=2, dh=64, P=16, count=120), (2, False, 4, True, 0)),
    (dict(lens=[(16 * 140, 1), (40, 2)], heads=40, kvh=2, dh=128, P=16, count=120), (2, False, 4, True, 0)),
    # tiles over lists by four waves, in the batch's order and with the longest contexts first
    (dict(lens=[(16 * 60 + 3, 200)], heads=32, kvh=8, dh=64, P=16, count=32), (1, True, 4, False, 0)),
    (dict(lens=[(16 * 60 + 3, 90), (5, 60), (300, 50)], heads=32, kvh=8, dh=64, P=16, count=32), (1, True, 4, False, 1)),
    (dict(lens=[(64 * 20 + 3, 220)], heads=32, kvh=8, dh=64, P=64, count=8), (1, True, 4, False, 0)),
    (dict(lens=[(16 * 60 + 3, 90), (5, 60), (300, 50)], heads=32, kvh=8, dh=128, P=16, count=16), (1, True, 4, False, 1)),
    (dict(lens=[(64 * 20 + 3, 90), (5, 60)], heads=40, kvh=8, dh=128, P=64, count=16), (1, True, 4, False, 1)),
    # by eight
    (dict(lens=[(16 * 60 + 3, 200)], heads=16, kvh=8, dh=64, P=16, count=32), (1, True, 8, False, 0)),
    (dict(lens=[(64 * 20 + 3, 90), (5, 50), (300, 42)], heads=24, kvh=8, dh=64, P=64, count=9), (1, True, 8, False, 1)),
    # a list a block, by eight and by four waves
    (dict(lens=[(64 * 20 + 3, 1), (5, 2)], heads=12, kvh=4, dh=64, P=64, count=9), (1, False, 8, False, 0)),
    (dict(lens=[(16 * 40 + 3, 5)], heads=6, kvh=2, dh=64, P=16, count=9), (1, False, 8, False, 0)),
    (dict(lens=[(64 * 20 + 3, 1), (5, 2)], heads=12, kvh=4, dh=128, P=64, count=9), (1, False, 4, False, 0)),
    (dict(lens=[(64 * 20 + 3, 1), (5, 2)], heads=40, kvh=2, dh=64, P=64, count=9), (2, False, 4, False, 0)),
    (dict(lens=[(64 * 60 + 3, 1), (5, 2)], heads=4, kvh=4, dh=64, P=64, count=50), (1, False, 4, True, 0)),
]


def attend_kind(form):
    return form[0], form[1] > 1, form[2], form[3] > 1, form[4]


def copy_form(pages, layers, kvh, dh, P):
    """(past the caches, sides a block) of a copy of so many pages"""
    cache = _cache(kvh, dh, P)
    pool = _lib.Kv8Pool((_lib.Kv8Cache * layers)(*[cache] * layers), None, AT, layers)
    return _form(2, lib.ane_debug_kv8_copy_form, pool, pages)


# Copies of so many pages, and whether they go past the caches: sides of 16 KB and more one a block, smaller ones
# several.
COPY = [
    (dict(pages=3500, layers=2, kvh=4, dh=64, P=64), (1, 1)),
    (dict(pages=400, layers=3, kvh=4, dh=128, P=256), (1, 1)),
    (dict(pages=5000, layers=5, kvh=2, dh=64, P=32), (1, 4)),
    (dict(pages=34000, layers=3, kvh=1, dh=64, P=16), (1, 6)),
    (dict(pages=2000, layers=2, kvh=4, dh=64, P=64), (0, 1)),
    (dict(pages=9000, layers=3, kvh=1, dh=64, P=16), (0, 6)),
]


def beam_form(requests, beams, vocab, half, hist, **_):
    """(loads of a wave, threads of the second launch, histories in a launch of their own)"""
    return _form(3, lib.ane_debug_beam_form, requests, beams, vocab, int(half), hist or 0)


BEAMS = [
    # four loads a wave: many fp32 logits, rows that end in a turn's first, second and third entry and elsewhere
    (dict(requests=34, beams=8, vocab=32003, half=False, hist=40, eos=32002, masked=0.5), (4, 512, 0)),
    (dict(requests=17, beams=16, vocab=32769, half=False, hist=None), (4, 1024, 0)),
    (dict(requests=1025, beams=4, vocab=2049, half=False, hist=9, eos=2048), (4, 512, 0)),
    (dict(requests=257, beams=16, vocab=2050, half=False, hist=600, eos=2049, masked=0.9), (4, 1024, 0)),
    (dict(requests=5461, beams=1, vocab=2051, half=False, hist=3, eos=0), (4, 512, 0)),
    (dict(requests=129, beams=32, vocab=2560, half=False, hist=5, eos=1), (4, 1024, 0)),
    (dict(requests=2049, beams=8, vocab=513, half=False, hist=17), (4, 512, 0)),
    (dict(requests=256, beams=2, vocab=16700, half=False, hist=4200, eos=3, wide=5), (4, 512, 0)),
    # below that line
    (dict(requests=1, beams=4, vocab=32000, half=False, hist=300, eos=2), (2, 512, 0)),
    # fp16: histories read ahead, moved by the second launch, in one of their own
    (dict(requests=34, beams=8, vocab=32003, half=True, hist=40, eos=32002), (2, 512, 0)),
    (dict(requests=3, beams=4, vocab=700, half=True, hist=2600, eos=3), (2, 512, 0)),
    (dict(requests=3, beams=16, vocab=700, half=True, hist=600, eos=3), (2, 1024, 0)),
    (dict(requests=2, beams=16, vocab=700, half=True, hist=4300, eos=3, wide=3), (2, 1024, 1)),
    (dict(requests=2, beams=5, vocab=700, half=True, hist=9000, wide=3), (2, 512, 1)),
]
