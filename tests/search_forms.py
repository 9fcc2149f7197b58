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
