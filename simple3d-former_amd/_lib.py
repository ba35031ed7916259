"""ctypes binding of libs3d_hip.so (C ABI: include/s3d_hip.h).

The struct mirrors are generated by parsing the public header, and checked against the library's own
`s3d_sizeof()` at load time, so the Python side cannot silently drift from the C side.  There is no fallback:
if the shared library is missing or an entry point fails, a RuntimeError is raised."""
import ctypes
import os
import re

_HERE = os.path.dirname(os.path.abspath(__file__))
_ROOT = os.path.dirname(_HERE)
# S3D_LIB_PATH: a differently-built libs3d_hip (e.g. the timeline debug build of csrc/Makefile TL=1); never a fallback
LIB_PATH = os.environ.get('S3D_LIB_PATH') or os.path.join(_HERE, 'libs3d_hip.so')
HEADER_PATH = os.path.join(_ROOT, 'include', 's3d_hip.h')

_SCALARS = {'int': ctypes.c_int, 'long': ctypes.c_long, 'float': ctypes.c_float, 'size_t': ctypes.c_size_t,
            'unsigned int': ctypes.c_uint, 'unsigned': ctypes.c_uint}


def _strip_comments(text):
    text = re.sub(r'/\*.*?\*/', ' ', text, flags=re.S)
    return re.sub(r'//[^\n]*', ' ', text)


def parse_structs(header_text):
    """{struct name: [(field, ctype), ...]} for every `typedef struct X {...} X;` of the header."""
    out = {}
    text = _strip_comments(header_text)
    for m in re.finditer(r'typedef\s+struct\s+(\w+)\s*\{(.*?)\}\s*(\w+)\s*;', text, flags=re.S):
        fields = []
        for decl in m.group(2).split(';'):
            decl = decl.strip()
            if not decl:
                continue
            first, *rest = [d.strip() for d in decl.split(',')]
            toks = first.replace('*', ' * ').split()
            name = toks[-1]
            base = [t for t in toks[:-1] if t not in ('const', '*')]
            is_ptr = '*' in toks[:-1]
            base_t = ' '.join(base)
            entries = [(name, is_ptr)]
            for r in rest:
                r = r.strip()
                entries.append((r.lstrip('* ').strip(), r.startswith('*')))
            for fname, ptr in entries:
                if ptr:
                    fields.append((fname, ctypes.c_void_p))
                else:
                    if base_t not in _SCALARS:
                        raise ValueError(f'unsupported scalar type {base_t!r} in {m.group(1)}.{fname}')
                    fields.append((fname, _SCALARS[base_t]))
        out[m.group(1)] = fields
    return out


def parse_functions(header_text):
    text = _strip_comments(header_text)
    return re.findall(r'\b(s3d_\w+)\s*\(', text)


_RET = {'int': ctypes.c_int, 'long': ctypes.c_long, 'size_t': ctypes.c_size_t, 'double': ctypes.c_double, 'float': ctypes.c_float,
        'void': None}


def parse_prototypes(header_text):
    """{function: (restype, [argtypes])} for every `T s3d_x(args);` of the header.  Pointers (and s3d_stream_t) become c_void_p -- torch
    data_ptr() ints, byref(struct), ctypes arrays and None all pass -- scalars their exact C type, so that a `long` / `size_t` / `double`
    argument handed over as a bare Python int or float is converted at full width (ctypes' default for an int is 32 bits)."""
    text = _strip_comments(header_text)
    out = {}
    for stmt in text.replace('}', ';').replace('{', ';').split(';'):
        m = re.match(r'\s*((?:const\s+)?[A-Za-z_][\w ]*?[\w\*])\s*\b(s3d_\w+)\s*\(([^()]*)\)\s*$', stmt, flags=re.S)
        if not m:
            continue
        ret, name, args = m.group(1).strip(), m.group(2), m.group(3).strip()
        if ret.startswith('typedef') or ret.startswith('extern'):
            continue
        if '*' in ret:
            restype = ctypes.c_char_p if 'char' in ret else ctypes.c_void_p
        else:
            restype = _RET[ret.replace('const', '').strip()]
        argtypes = []
        if args and args != 'void':
            for a in args.split(','):
                a = ' '.join(a.split())
                if '*' in a or 's3d_stream_t' in a:
                    argtypes.append(ctypes.c_char_p if re.match(r'const char\s*\*\s*\w*$', a) else ctypes.c_void_p)
                    continue
                toks = [t for t in a.split() if t != 'const']
                base = ' '.join(toks[:-1]) if len(toks) > 1 else toks[0]
                if base == 'double':
                    argtypes.append(ctypes.c_double)
                elif base in _SCALARS:
                    argtypes.append(_SCALARS[base])
                else:
                    raise ValueError(f'unsupported parameter type {a!r} in {name}')
        out[name] = (restype, argtypes)
    return out


with open(HEADER_PATH) as _f:
    _HEADER = _f.read()
_STRUCT_FIELDS = parse_structs(_HEADER)
DECLARED_FUNCTIONS = sorted(set(parse_functions(_HEADER)) - {'s3d_stream_t'})
PROTOTYPES = parse_prototypes(_HEADER)


def _make_struct(name, fields):
    return type(name, (ctypes.Structure,), {'_fields_': fields})


STRUCTS = {n: _make_struct(n, f) for n, f in _STRUCT_FIELDS.items()}
globals().update(STRUCTS)

_lib = None


def lib():
    """Loads libs3d_hip.so once; raises RuntimeError (never falls back) if it is absent or inconsistent."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(f'{LIB_PATH} is missing: build it with `python -c "import __graft_entry__ as g; g.build()"` '
                           f'(hipcc --offload-arch=gfx950).  The HIP path has no CPU fallback.')
    try:
        L = ctypes.CDLL(LIB_PATH)
    except OSError as e:
        raise RuntimeError(f'cannot load {LIB_PATH}: {e}') from e
    L.s3d_last_error_string.restype = ctypes.c_char_p
    L.s3d_sizeof.restype = ctypes.c_size_t
    L.s3d_sizeof.argtypes = [ctypes.c_char_p]
    # entry points that do not return int (ctypes' default restype would truncate a > 2 GiB workspace size)
    for fn, rt in (('s3d_block_workspace_bytes', ctypes.c_size_t), ('s3d_block_wgrad_slot_bytes', ctypes.c_size_t),
                   ('s3d_cov_collect', ctypes.c_long), ('s3d_prof_skip_get', ctypes.c_double)):
        if hasattr(L, fn):
            getattr(L, fn).restype = rt
    for fn in DECLARED_FUNCTIONS:
        if not hasattr(L, fn):
            raise RuntimeError(f'{LIB_PATH} does not export {fn} declared in include/s3d_hip.h')
    # every prototype of the header becomes restype + argtypes (a size_t / long / double passed as a bare Python
    # number would otherwise travel as a 32-bit int)
    missing = set(DECLARED_FUNCTIONS) - set(PROTOTYPES)
    if missing:
        raise RuntimeError(f'include/s3d_hip.h: could not parse the prototypes of {sorted(missing)}')
    for fn, (rt, at) in PROTOTYPES.items():
        f = getattr(L, fn)
        f.restype = rt
        f.argtypes = at
    for n, S in STRUCTS.items():
        c = L.s3d_sizeof(n.encode())
        if c != ctypes.sizeof(S):
            raise RuntimeError(f'ABI mismatch for {n}: header mirror {ctypes.sizeof(S)} B, library {c} B')
    _lib = L
    return L


def check(rc, what=''):
    if rc != 0:
        msg = lib().s3d_last_error_string().decode(errors='replace')
        raise RuntimeError(f's3d {what} failed (rc={rc}): {msg}')


def ptr(t):
    """Device pointer of a torch tensor (or None)."""
    if t is None:
        return None
    return ctypes.c_void_p(t.data_ptr())


def fill(struct, **kw):
    """Assigns fields of a ctypes struct from tensors / numbers (tensors -> data_ptr)."""
    names = {f[0] for f in struct._fields_}
    for k, v in kw.items():
        if k not in names:
            raise AttributeError(f'{type(struct).__name__} has no field {k}')
        if hasattr(v, 'data_ptr'):
            v = v.data_ptr()
        setattr(struct, k, v)
    return struct


_current = None


def current_stream():
    """The current HIP stream of the current device.  torch.cuda.current_stream() builds a Stream object (2.7 us a call); the raw handle is the
    same value."""
    global _current
    if _current is None:
        import torch
        raw = getattr(torch._C, '_cuda_getCurrentRawStream', None)
        device = torch.cuda.current_device
        _current = (lambda: raw(device())) if raw is not None else (lambda: torch.cuda.current_stream().cuda_stream)
    return ctypes.c_void_p(_current())
