"""The C header and the binding notes at the repository root name the same surface: every function include/bm_moe.h
declares appears in the notes' extern "C" block with the same number of arguments under the same names, in the same
order, and the block binds nothing the header does not declare. (That the built library exports every declared symbol is
test_capi_cpu.py's part.)"""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NOTES = os.path.join(ROOT, "INTEGRATION.md")


def header_functions():
    src = open(os.path.join(ROOT, "include", "bm_moe.h")).read()
    src = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
    src = re.sub(r"^\s*#.*$", "", src, flags=re.M)
    src = re.sub(r"typedef struct \w+ \{.*?\} \w+;", "", src, flags=re.S)
    out = {}
    for name, params in re.findall(r"\b(bm_\w+)\s*\(([^;{}]*?)\)\s*;", src, flags=re.S):
        params = " ".join(params.split())
        names = [] if params in ("", "void") else [re.search(r"(\w+)$", p.strip()).group(1) for p in params.split(",")]
        assert name not in out, f"{name} declared twice"
        out[name] = names
    return out


def bound_functions():
    text = open(NOTES).read()
    block = re.search(r'extern "C" \{(.*?)\n\}', text, flags=re.S).group(1)
    out = {}
    for name, params in re.findall(r"pub fn (bm_\w+)\s*\((.*?)\)\s*(?:->[^;]*)?;", block, flags=re.S):
        params = " ".join(params.split())
        names = [] if not params else [p.split(":")[0].strip() for p in params.split(",")]
        assert name not in out, f"{name} bound twice"
        out[name] = names
    return out


def test_every_declared_function_is_bound_with_the_same_arguments():
    declared, bound = header_functions(), bound_functions()
    assert len(declared) > 60
    assert sorted(set(declared) - set(bound)) == [], "declared in include/bm_moe.h, missing from the binding notes"
    assert sorted(set(bound) - set(declared)) == [], "bound in the notes, not declared in include/bm_moe.h"
    for name, names in declared.items():
        assert bound[name] == names, f"{name}: the header has ({', '.join(names)}), the binding ({', '.join(bound[name])})"


def test_the_build_recipe_names_every_source_of_the_library():
    """The build.rs shown compiles what the Makefile compiles."""
    mk = open(os.path.join(ROOT, "bloomery_amd", "csrc", "Makefile")).read()
    srcs = re.search(r"^SRCS = (.*)$", mk, flags=re.M).group(1).split()
    text = open(NOTES).read()
    recipe = re.search(r"## build\.rs(.*?)## extern", text, flags=re.S).group(1)
    assert len(srcs) >= 7
    for s in srcs:
        assert f'"{s}"' in recipe, f"{s} is built by the Makefile and missing from the build.rs shown"


# what Rust takes for no plain identifier (strict and reserved words)
RUST_WORDS = set("""as break const continue crate else enum extern false fn for if impl in let loop match mod move mut pub ref return self Self static
struct super trait true type unsafe use where while async await dyn abstract become box do final macro override priv typeof unsized virtual
yield try gen""".split())
RUST_TYPE = re.compile(r"(\*(const|mut) )*(c_int|c_char|c_void|usize|[iu](8|16|32|64)|f32|f64|bool|bm_\w+)$")


def test_the_binding_block_is_rust():
    """A name that is a word of the language's own, in one declaration, costs the whole block: names of functions, arguments and fields, and
    the types of arguments and results, in every Rust block of the notes."""
    blocks = re.findall(r"```rust\n(.*?)```", open(NOTES).read(), flags=re.S)
    assert blocks
    block = "\n".join(blocks)
    for name in re.findall(r"pub (?:const |static |fn |struct )?(r#\w+|\w+)\s*[:({=]", block):
        assert name not in RUST_WORDS, name
    functions = re.findall(r"pub fn (bm_\w+)\s*\((.*?)\)\s*(?:->\s*([^;]*?))?\s*;", block, flags=re.S)
    assert len(functions) > 60
    for name, params, result in functions:
        assert not result or RUST_TYPE.match(" ".join(result.split())), (name, result)
        for p in filter(None, (" ".join(p.split()) for p in params.split(","))):
            arg, of = (t.strip() for t in p.split(":", 1))
            assert re.fullmatch(r"(r#)?[a-z_]\w*", arg) and arg not in RUST_WORDS, f"{name}: {arg} is no name of an argument"
            assert RUST_TYPE.match(of), (name, p)
