{===============================================================================
  Gemma4.Beam - binding of libgemma4_sampler.so's beam search and page cache
  (include/gemma4_beam.h), beside Gemma4.Sampler.

  Where TModel.Generate (src/Gemma4.Model.pas:2829-2938) draws one token, a
  search keeps several token strings per sequence.  As in Gemma4.Sampler, every
  external has its export's argument order and C types, arrays and records are
  typed pointers passed by value, and a failing call of the classes adds an
  esError entry to GetErrors() and returns False.
===============================================================================}

unit Gemma4.Beam;

{$IFDEF FPC}{$MODE DELPHI}{$ENDIF}

interface

uses
  SysUtils,
  StdApp.Base,
  Gemma4.Sampler;

const
  CSM_ERR_BEAM = 'SM05';
  CSM_ERR_PAGES = 'SM06';

  G4S_BEAM_MAX_BEAMS = 64;
  G4S_BEAM_MAX_ROWS = 65535;
  G4S_PAGES_MAX_ROWS = 2048;
  G4S_PAGES_MAX_PAGES = 1048576;

type
  { PG4SBeam, PG4SPages }
  // opaque g4s_beam* and g4s_pages*
  PG4SBeam = Pointer;
  PPG4SBeam = ^PG4SBeam;
  PG4SPages = Pointer;
  PPG4SPages = ^PG4SPages;

  { TG4SPageGeometry }
  // g4s_page_geometry: page g of plane p at p*PlaneStride + g*PageStride
  // bytes of the pool
  TG4SPageGeometry = record
    PageTokens: Integer;
    NPages: Integer;
    MaxRows: Integer;
    MaxSlots: Integer;
    Planes: Integer;
    Parts: Integer;
    TokenBytes: Int64;
    PlaneStride: Int64;
    PageStride: Int64;
  end;
  PG4SPageGeometry = ^TG4SPageGeometry;

  { TG4SPageState }
  // g4s_page_state: GPU arrays of a state
  TG4SPageState = record
    Table: PInteger;
    Lengths: PInteger;
    Refs: PInteger;
  end;
  PG4SPageState = ^TG4SPageState;

  { TG4SBeamConfig }
  TG4SBeamConfig = record
    Beams: Integer;
    MaxTokens: Integer;
    NBest: Integer;
    EarlyStop: Integer;
    LengthPenalty: Single;
  end;
  PG4SBeamConfig = ^TG4SBeamConfig;

  { TG4SBeamStates }
  TG4SBeamStates = record
    DState: Pointer;
    Planes: Int64;
    PlaneStride: Int64;
    RowStride: Int64;
    RowBytes: Int64;
  end;
  PG4SBeamStates = ^TG4SBeamStates;

  { TG4SBeamCache }
  TG4SBeamCache = record
    Pages: PG4SPages;
    States: array[0..1] of TG4SPageState;
    DPool: Pointer;
  end;
  PG4SBeamCache = ^TG4SBeamCache;

  { TG4SBeamStep }
  // what the model step gets; Tokens and Parents are host arrays
  TG4SBeamStep = record
    Tokens: PInteger;
    Parents: PInteger;
    DTokens: PInteger;
    DParents: PInteger;
    Rows: Integer;
    State: Integer;
  end;
  PG4SBeamStep = ^TG4SBeamStep;

  TG4SBeamForwardFn = function(AUser: Pointer; AStep: PG4SBeamStep): Integer; cdecl;

function g4s_beam_create(AOut: PPG4SBeam; AVocab: Integer; AMaxBatch: Integer;
  AMaxBeams: Integer; ASoftcap: Single; AHipStream: Pointer): Integer; cdecl;
  external CG4SLib;
function g4s_beam_destroy(ABeam: PG4SBeam): Integer; cdecl; external CG4SLib;
function g4s_beam_last_error(ABeam: PG4SBeam): PAnsiChar; cdecl; external CG4SLib;
function g4s_beam_select(ABeam: PG4SBeam; ADevLogits: Pointer; ADType: Integer;
  ARowStride: Int64; ABatch: Integer; ABeams: Integer; ADevScores: PSingle;
  ANSelect: Integer; ADevParents: PInteger; ADevTokens: PInteger; ADevOut: PSingle;
  ADevLse: PSingle): Integer; cdecl; external CG4SLib;
function g4s_beam_reorder(ABeam: PG4SBeam; ADevSrc: Pointer; ADevDst: Pointer;
  APlanes: Int64; APlaneStride: Int64; ABatch: Integer; ABeams: Integer;
  ARowStride: Int64; ARowBytes: Int64; ADevParents: PInteger): Integer; cdecl;
  external CG4SLib;
function g4s_pages_create(AOut: PPG4SPages; AGeometry: PG4SPageGeometry;
  AHipStream: Pointer): Integer; cdecl; external CG4SLib;
function g4s_pages_destroy(APages: PG4SPages): Integer; cdecl; external CG4SLib;
function g4s_pages_last_error(APages: PG4SPages): PAnsiChar; cdecl; external CG4SLib;
function g4s_pages_advance(APages: PG4SPages; AFrom: PG4SPageState; AFromRows: Integer;
  ATo: PG4SPageState; ARows: Integer; ADevParents: PInteger; ADevGrow: PInteger;
  ADevPool: Pointer; ADevStatus: PInteger): Integer; cdecl; external CG4SLib;
function g4s_pages_compact(APages: PG4SPages; AFrom: PG4SPageState; ATo: PG4SPageState;
  ARows: Integer; ADevPool: Pointer; ADevStatus: PInteger): Integer; cdecl;
  external CG4SLib;
function g4s_pages_copy(APages: PG4SPages; ADevSrcPool: Pointer; ADevDstPool: Pointer;
  AN: Integer; ADevSrcPages: PInteger; ADevDstPages: PInteger;
  ADevTokens: PInteger): Integer; cdecl; external CG4SLib;
function g4s_beam_generate(ABeam: PG4SBeam; ABatch: Integer; AConfig: PG4SBeamConfig;
  ADevLogits: Pointer; ADType: Integer; ARowStride: Int64; AStates: PG4SBeamStates;
  ACache: PG4SBeamCache; AForward: TG4SBeamForwardFn; AUser: Pointer; ATokens: PInteger;
  ALengths: PInteger; AScores: PSingle): Integer; cdecl; external CG4SLib;

type
  { TGpuBeamSearch }
  TGpuBeamSearch = class(TBaseObject)
  private
    FHandle: PG4SBeam;
    FVocab: Integer;
    function Fail(const AStatus: Integer): Boolean;
  public
    destructor Destroy(); override;

    // g4s_beam_create: the whole workspace is allocated here
    function Open(const AVocab: Integer; const AMaxBatch: Integer;
      const AMaxBeams: Integer; const ASoftcap: Single;
      const AHipStream: Pointer = nil): Boolean;
    procedure Close();

    // the search around the engine's forward pass; AConfig^.NBest results
    // per sequence.  ARowStride: elements from row to row of ADevLogits, 0 = the
    // vocabulary; rows start on multiples of 16 bytes
    function Generate(const ABatch: Integer; const AConfig: PG4SBeamConfig;
      const ADevLogits: Pointer; const ADType: Integer; const AStates: PG4SBeamStates;
      const ACache: PG4SBeamCache; const AForward: TG4SBeamForwardFn;
      const AUser: Pointer; const ATokens: PInteger; const ALengths: PInteger;
      const AScores: PSingle; const ARowStride: Int64 = 0): Boolean;

    function LastError(): string;

    property Handle: PG4SBeam read FHandle;
  end;

  { TGpuPageCache }
  TGpuPageCache = class(TBaseObject)
  private
    FHandle: PG4SPages;
    function Fail(const AStatus: Integer): Boolean;
  public
    destructor Destroy(); override;
    function Open(const AGeometry: PG4SPageGeometry;
      const AHipStream: Pointer = nil): Boolean;
    procedure Close();
    function LastError(): string;
    property Handle: PG4SPages read FHandle;
  end;

implementation

{ TGpuBeamSearch }

destructor TGpuBeamSearch.Destroy();
begin
  Close();
  inherited;
end;

function TGpuBeamSearch.LastError(): string;
begin
  Result := string(AnsiString(g4s_beam_last_error(FHandle)));
end;

function TGpuBeamSearch.Fail(const AStatus: Integer): Boolean;
begin
  GetErrors().Add(esError, CSM_ERR_BEAM, 'Beam search status %d: %s', [AStatus, LastError()]);
  Result := False;
end;

function TGpuBeamSearch.Open(const AVocab: Integer; const AMaxBatch: Integer;
  const AMaxBeams: Integer; const ASoftcap: Single; const AHipStream: Pointer): Boolean;
var
  LStatus: Integer;
  LHandle: PG4SBeam;
begin
  Close();
  LHandle := nil;
  LStatus := g4s_beam_create(@LHandle, AVocab, AMaxBatch, AMaxBeams, ASoftcap, AHipStream);
  if LStatus <> G4S_OK then
    Exit(Fail(LStatus));
  FHandle := LHandle;
  FVocab := AVocab;
  Result := True;
end;

procedure TGpuBeamSearch.Close();
begin
  if FHandle <> nil then
  begin
    g4s_beam_destroy(FHandle);
    FHandle := nil;
  end;
end;

function TGpuBeamSearch.Generate(const ABatch: Integer; const AConfig: PG4SBeamConfig;
  const ADevLogits: Pointer; const ADType: Integer; const AStates: PG4SBeamStates;
  const ACache: PG4SBeamCache; const AForward: TG4SBeamForwardFn; const AUser: Pointer;
  const ATokens: PInteger; const ALengths: PInteger; const AScores: PSingle;
  const ARowStride: Int64): Boolean;
var
  LStatus: Integer;
  LRowStride: Int64;
begin
  LRowStride := ARowStride;
  if LRowStride = 0 then
    LRowStride := FVocab;
  LStatus := g4s_beam_generate(FHandle, ABatch, AConfig, ADevLogits, ADType, LRowStride,
    AStates, ACache, AForward, AUser, ATokens, ALengths, AScores);
  if LStatus <> G4S_OK then
    Exit(Fail(LStatus));
  Result := True;
end;

{ TGpuPageCache }

destructor TGpuPageCache.Destroy();
begin
  Close();
  inherited;
end;

function TGpuPageCache.LastError(): string;
begin
  Result := string(AnsiString(g4s_pages_last_error(FHandle)));
end;

function TGpuPageCache.Fail(const AStatus: Integer): Boolean;
begin
  GetErrors().Add(esError, CSM_ERR_PAGES, 'Page cache status %d: %s', [AStatus, LastError()]);
  Result := False;
end;

function TGpuPageCache.Open(const AGeometry: PG4SPageGeometry;
  const AHipStream: Pointer): Boolean;
var
  LStatus: Integer;
  LHandle: PG4SPages;
begin
  Close();
  LHandle := nil;
  LStatus := g4s_pages_create(@LHandle, AGeometry, AHipStream);
  if LStatus <> G4S_OK then
    Exit(Fail(LStatus));
  FHandle := LHandle;
  Result := True;
end;

procedure TGpuPageCache.Close();
begin
  if FHandle <> nil then
  begin
    g4s_pages_destroy(FHandle);
    FHandle := nil;
  end;
end;

end.
