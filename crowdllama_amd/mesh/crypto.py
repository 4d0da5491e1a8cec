"""Cryptographic identity and encrypted transport for the mesh.

The reference gets peer identity and channel security from libp2p: ed25519
peer keys (reference internal/keys/keys.go:38-98) and noise/TLS stream
encryption negotiated by the host (reference
internal/discovery/discovery.go:48-84, go.mod:8). This module provides the
MI355X-native mesh's equivalent with no third-party dependencies (the
build environment has no `cryptography`/`nacl` wheels):

- ed25519 signatures (RFC 8032) — peer identity keys; Resource records and
  handshakes are signed and verified.
- X25519 Diffie-Hellman (RFC 7748) — per-connection ephemeral key
  agreement (forward secrecy).
- A SIGMA-style authenticated handshake binding the ephemeral exchange to
  both ed25519 identities; peer_id = hash of the ed25519 public key, so a
  dialer that knows a peer_id cryptographically verifies it is talking to
  that peer.
- An encrypt-then-MAC secure channel over the existing 4-byte length
  framing: per-direction keys from BLAKE2b-HKDF, BLAKE2b keystream in
  counter mode, BLAKE2b-128 MAC, strictly increasing per-frame counters
  (replay/reorder rejection).

Implementation note: the field/curve arithmetic is written from RFC
8032/7748 pseudocode (these are public algorithms); Python's bignums make
the schoolbook form practical (~1-5 ms per operation — handshake cost is
per-connection, not per-token). BLAKE2b comes from hashlib (C speed).
"""

from __future__ import annotations

import hashlib
import hmac
import os
import struct

# ---------------------------------------------------------------- ed25519
# RFC 8032 (Ed25519). Little-endian encodings throughout.

_P = 2**255 - 19
_L = 2**252 + 27742317777372353535851937790883648493
_D = (-121665 * pow(121666, _P - 2, _P)) % _P
_I = pow(2, (_P - 1) // 4, _P)


def _sha512(*parts: bytes) -> bytes:
    h = hashlib.sha512()
    for p in parts:
        h.update(p)
    return h.digest()


def _inv(x: int) -> int:
    return pow(x, _P - 2, _P)


def _recover_x(y: int, sign: int) -> int:
    if y >= _P:
        raise ValueError("bad point")
    x2 = (y * y - 1) * _inv(_D * y * y + 1) % _P
    if x2 == 0:
        if sign:
            raise ValueError("bad point")
        return 0
    x = pow(x2, (_P + 3) // 8, _P)
    if (x * x - x2) % _P != 0:
        x = x * _I % _P
    if (x * x - x2) % _P != 0:
        raise ValueError("bad point")
    if (x & 1) != sign:
        x = _P - x
    return x


# extended homogeneous coordinates (X, Y, Z, T), x = X/Z, y = Y/Z, xy = T/Z
_G_Y = 4 * _inv(5) % _P
_G_X = _recover_x(_G_Y, 0)
_ID = (0, 1, 1, 0)


def _pt_add(p, q):
    X1, Y1, Z1, T1 = p
    X2, Y2, Z2, T2 = q
    a = (Y1 - X1) * (Y2 - X2) % _P
    b = (Y1 + X1) * (Y2 + X2) % _P
    c = 2 * T1 * T2 * _D % _P
    d = 2 * Z1 * Z2 % _P
    e, f, g, h = b - a, d - c, d + c, b + a
    return (e * f % _P, g * h % _P, f * g % _P, e * h % _P)


def _pt_mul(s: int, p):
    q = _ID
    while s > 0:
        if s & 1:
            q = _pt_add(q, p)
        p = _pt_add(p, p)
        s >>= 1
    return q


def _pt_eq(p, q) -> bool:
    X1, Y1, Z1, _ = p
    X2, Y2, Z2, _ = q
    return (X1 * Z2 - X2 * Z1) % _P == 0 and (Y1 * Z2 - Y2 * Z1) % _P == 0


def _pt_compress(p) -> bytes:
    X, Y, Z, _ = p
    zi = _inv(Z)
    x, y = X * zi % _P, Y * zi % _P
    return int.to_bytes(y | ((x & 1) << 255), 32, "little")


def _pt_decompress(b: bytes):
    if len(b) != 32:
        raise ValueError("bad point length")
    n = int.from_bytes(b, "little")
    sign = n >> 255
    y = n & ((1 << 255) - 1)
    x = _recover_x(y, sign)
    return (x, y, 1, x * y % _P)


_G = (_G_X, _G_Y, 1, _G_X * _G_Y % _P)


def _clamp(h: bytes) -> int:
    a = int.from_bytes(h[:32], "little")
    a &= (1 << 254) - 8
    a |= 1 << 254
    return a


def ed25519_public(seed: bytes) -> bytes:
    """Public key (32 B) for a 32-byte private seed."""
    if len(seed) != 32:
        raise ValueError("seed must be 32 bytes")
    a = _clamp(_sha512(seed))
    return _pt_compress(_pt_mul(a, _G))


def ed25519_sign(seed: bytes, msg: bytes) -> bytes:
    """RFC 8032 signature (64 B)."""
    h = _sha512(seed)
    a = _clamp(h)
    pub = _pt_compress(_pt_mul(a, _G))
    r = int.from_bytes(_sha512(h[32:], msg), "little") % _L
    R = _pt_compress(_pt_mul(r, _G))
    k = int.from_bytes(_sha512(R, pub, msg), "little") % _L
    s = (r + k * a) % _L
    return R + int.to_bytes(s, 32, "little")


def ed25519_verify(pub: bytes, msg: bytes, sig: bytes) -> bool:
    """True iff sig is a valid signature of msg under pub."""
    try:
        if len(sig) != 64 or len(pub) != 32:
            return False
        A = _pt_decompress(pub)
        R = _pt_decompress(sig[:32])
        s = int.from_bytes(sig[32:], "little")
        if s >= _L:
            return False
        k = int.from_bytes(_sha512(sig[:32], pub, msg), "little") % _L
        return _pt_eq(_pt_mul(s, _G), _pt_add(R, _pt_mul(k, A)))
    except (ValueError, OverflowError):
        return False


# ---------------------------------------------------------------- X25519
# RFC 7748 montgomery-ladder scalar multiplication.

_A24 = 121665


def _x25519_scalar(k_bytes: bytes) -> int:
    k = bytearray(k_bytes)
    k[0] &= 248
    k[31] &= 127
    k[31] |= 64
    return int.from_bytes(bytes(k), "little")


def x25519(k_bytes: bytes, u_bytes: bytes) -> bytes:
    """Scalar multiplication on curve25519 (RFC 7748 §5)."""
    k = _x25519_scalar(k_bytes)
    u = int.from_bytes(u_bytes, "little") & ((1 << 255) - 1)
    x1, x2, z2, x3, z3 = u, 1, 0, u, 1
    swap = 0
    for t in range(254, -1, -1):
        kt = (k >> t) & 1
        swap ^= kt
        if swap:
            x2, x3 = x3, x2
            z2, z3 = z3, z2
        swap = kt
        a = (x2 + z2) % _P
        aa = a * a % _P
        b = (x2 - z2) % _P
        bb = b * b % _P
        e = (aa - bb) % _P
        c = (x3 + z3) % _P
        d = (x3 - z3) % _P
        da = d * a % _P
        cb = c * b % _P
        x3 = (da + cb) % _P
        x3 = x3 * x3 % _P
        z3 = (da - cb) % _P
        z3 = u * z3 * z3 % _P
        x2 = aa * bb % _P
        z2 = e * (aa + _A24 * e) % _P
    if swap:
        x2, x3 = x3, x2
        z2, z3 = z3, z2
    return int.to_bytes(x2 * pow(z2, _P - 2, _P) % _P, 32, "little")


_X25519_BASE = int.to_bytes(9, 32, "little")


def x25519_public(priv: bytes) -> bytes:
    return x25519(priv, _X25519_BASE)


# ------------------------------------------------------------ kdf / cipher

def hkdf(ikm: bytes, info: bytes, n: int = 64, salt: bytes = b"") -> bytes:
    """HKDF-SHA256 (RFC 5869)."""
    prk = hmac.new(salt or b"\x00" * 32, ikm, hashlib.sha256).digest()
    out = b""
    t = b""
    i = 1
    while len(out) < n:
        t = hmac.new(prk, t + info + bytes([i]), hashlib.sha256).digest()
        out += t
        i += 1
    return out[:n]


def _keystream(key: bytes, nonce: bytes, n: int) -> bytes:
    """BLAKE2b-keyed PRF in counter mode (64 B per call; hashlib C speed).
    Standard PRF-as-stream-cipher construction; key/nonce never reused
    (per-frame counters below)."""
    out = bytearray()
    ctr = 0
    while len(out) < n:
        out += hashlib.blake2b(nonce + struct.pack("<Q", ctr), key=key,
                               digest_size=64).digest()
        ctr += 1
    return bytes(out[:n])


class SecureChannel:
    """Per-direction encrypt-then-MAC frame cipher with replay protection.

    seal(): ct = pt XOR keystream(k_enc, ctr); tag = BLAKE2b-128(k_mac,
    ctr || ct). open() enforces the counter (strictly sequential), so
    frames cannot be replayed, dropped or reordered undetected.
    """

    def __init__(self, k_send: bytes, k_recv: bytes):
        self._ks_enc = k_send[:32]
        self._ks_mac = k_send[32:]
        self._kr_enc = k_recv[:32]
        self._kr_mac = k_recv[32:]
        self._send_ctr = 0
        self._recv_ctr = 0

    def seal(self, pt: bytes) -> bytes:
        nonce = struct.pack("<Q", self._send_ctr)
        self._send_ctr += 1
        ct = bytes(a ^ b for a, b in
                   zip(pt, _keystream(self._ks_enc, nonce, len(pt))))
        tag = hashlib.blake2b(nonce + ct, key=self._ks_mac,
                              digest_size=16).digest()
        return ct + tag

    def open(self, frame: bytes) -> bytes:
        if len(frame) < 16:
            raise ValueError("short frame")
        ct, tag = frame[:-16], frame[-16:]
        nonce = struct.pack("<Q", self._recv_ctr)
        want = hashlib.blake2b(nonce + ct, key=self._kr_mac,
                               digest_size=16).digest()
        if not hmac.compare_digest(tag, want):
            raise ValueError("MAC verification failed")
        self._recv_ctr += 1
        return bytes(a ^ b for a, b in
                     zip(ct, _keystream(self._kr_enc, nonce, len(ct))))


# ------------------------------------------------------------- handshake

PROTO_TAG = b"cla-noise-v1"


def handshake_msg1(eph_priv: bytes, id_pub: bytes) -> bytes:
    """Initiator -> responder: ephemeral X25519 pub + ed25519 identity."""
    return x25519_public(eph_priv) + id_pub


def handshake_msg2(eph_priv: bytes, id_seed: bytes, id_pub: bytes,
                   msg1: bytes) -> bytes:
    """Responder -> initiator: its ephemeral + identity + signature over
    the transcript (binds the DH exchange to the responder identity)."""
    e_pub = x25519_public(eph_priv)
    sig = ed25519_sign(id_seed, PROTO_TAG + b"|resp|" + msg1 + e_pub + id_pub)
    return e_pub + id_pub + sig


def handshake_msg3(id_seed: bytes, msg1: bytes, msg2: bytes) -> bytes:
    """Initiator -> responder: signature over the transcript."""
    return ed25519_sign(id_seed, PROTO_TAG + b"|init|" + msg1 + msg2)


def derive_channels(eph_priv: bytes, peer_eph_pub: bytes, msg1: bytes,
                    msg2: bytes, initiator: bool) -> SecureChannel:
    shared = x25519(eph_priv, peer_eph_pub)
    km = hkdf(shared, PROTO_TAG + msg1 + msg2, 128)
    k_i, k_r = km[:64], km[64:]
    return SecureChannel(k_i, k_r) if initiator else SecureChannel(k_r, k_i)


def new_keypair() -> tuple[bytes, bytes]:
    """(seed, pub) ed25519 identity keypair."""
    seed = os.urandom(32)
    return seed, ed25519_public(seed)


def peer_id_from_pub(pub: bytes) -> str:
    """Stable peer id derived from the identity public key: any peer that
    knows an id can verify the key it is shown hashes to it (the reference
    gets the same property from libp2p multihash peer IDs)."""
    return "cla" + hashlib.sha256(b"cla-peer-id|" + pub).hexdigest()[:40]
